// Prompt attention over a paged cache on the sm_100a tensor cores (tcgen05 + TMEM), head_dim 64 or 128.
//
// One CTA owns two tiles of 128 query rows of one KV head, a row being a (token, head of the group) pair: short ragged
// prompts fill tiles, the causal triangle wastes 128 / group tokens instead of 128, and K and V are shared by the group.
// Per 128-row key tile and query tile t:
//
//   S_t  = Q_t K^T         tcgen05.mma kind::f16, 128 x 128 x D, accumulator in TMEM
//   P_t  = 2^(s - m)       one softmax thread per query row reads its row of S_t from TMEM and writes bf16 P_t back over
//                          it, 64 keys at a time: keys 0..63 into columns 0..31, keys 64..127 into columns 64..95, each
//                          over scores the thread has already read, so the two units need no hand-shake
//   O_t += P_t V           tcgen05.mma with the A operand in TMEM, one per unit and 16 keys; the first unit's products run
//                          while the second unit is exponentiated
//
// The running reference m of a row may lag its maximum by up to 2^40: a probability of 2^40 is as exact in bf16 P and in
// the f32 sums as one of 1 (P, O and l scale together). After a row's first unit no maximum is taken; the sum of a unit's
// probabilities tells when a score has outgrown m, and only then is the maximum found and O rescaled in TMEM. Key tiles
// run from the last one down: with a distance bias a row's largest scores lie at its own position, so m is right at once.
//
// Bound by the chain of a query tile: scores (512 cycles of the tensor pipe), the row's exponentials (128 at 8 cycles of the
// special-function unit), PV (512), and the hand-offs between them; two query tiles alternate, and TMEM (two score tiles and
// two outputs, 4 x 128 columns at D = 128) has no room for a third. Cycle counters at 8192 tokens: 3624 per key tile of both
// query tiles, of which the tensor pipe works 2048 and a group waits 1110 for its scores. Measured (32 query and 8 KV heads
// of 128): 462 us for 8192 tokens (1190 TFLOP/s of the pairs under the mask, 0.72 of the measured burst), 263 to 283 us for
// 2 x 515 tokens over 12000 rows, capped (751 to 808 TFLOP/s, by the machine), 111 us for 3 x 1600 tokens over NVFP4 pages with bias and prefix.
//
// Roles: warp 0 loads (TMA; boxes never cross a page), warp 1 issues, warps 4-7 and 8-11 are the softmax groups, a thread
// per row. Over NVFP4 pages warps 0, 2, 3 and 12 expand rows to bf16 into the same swizzled tiles (exact: code x scale has
// six significant bits), a tile ahead of the products.
//
// Blocks. cu_q and the lengths are on the device: CTA y-th block finds its sequence by counting blocks, KV heads run
// fastest (they share nothing, but the heads of a block end together), within a sequence the latest (longest) blocks
// start first. Where there are fewer blocks than SMs the key tiles of a block are cut over several CTAs, whose
// (m, l, O) a second kernel joins in order.
//
// The ordinary unit (every key seen, reference at hand) is kept apart from the general form: merged into one, the pass took
// 2226 cycles instead of 1586. Capped scores below the cap go through a polynomial (the FMA pipe) instead of two
// special-function operations each: 475 to 322 us at 2 x 515 tokens over 12000 rows.
//
// Every wait is bounded.
#include "paged.cuh"

#include <cuda_fp16.h>

#include <algorithm>

namespace {

using namespace tc5;

constexpr int BC = 128;                  // key rows per tile
constexpr int QT = 128;                  // query rows per tile, two tiles per CTA
constexpr int HALF = BC * 128;           // 64 features of a tile: 16 KB
constexpr int KSTAGES = 2, VSTAGES = 2;
constexpr int MAX_SPLITS = 16;
constexpr uint32_t MIN_SPLIT_TILES = 4;  // key tiles per CTA below which cutting further does not pay

struct PromptParams {
  CUtensorMap tmap_q;                    // [tokens, heads, D], box 64 x group x tile_tokens
  CUtensorMap tmap_k, tmap_v;            // bf16 pools
  PagedView c;
  const uint8_t *k, *v, *ks, *vs;        // NVFP4 pools
  __nv_bfloat16* out;
  const int32_t* cu_q;
  const float* slopes;
  int4* meta;                            // per block: first token, tokens, -, - (splits > 1)
  float* part;                           // [block][kv head][split][256][D + 4]
  uint32_t tokens, heads, group, tile_tokens, blocks, splits, box_rows;
  mb_fastdiv group_div;
  float scale_log2, cap_log2, inv_cap;   // inv_cap = scale / softcap, 0 without a cap
  int* flags;
};

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
// Two-lane f32 arithmetic of sm_100 (each lane an IEEE round-to-nearest op).
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 f2_pack(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_unpack(f32x2 v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ f32x2 f2_fma(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 f2_add(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 f2_mul(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// tanh of two values with |x| <= 1: x + x^3 q(x^2), q of degree four, off by 3.3e-7 and by 1.3e-6 of its value at most (a
// weighted least-squares fit, reweighted towards the smallest maximum). Without the two special-function operations of
// paged_tanh. The powers of c moved into the coefficients save an operation a pair and no time (263 us either way at 2 x 515
// tokens over 12000 rows); a shorter fit for units within half the cap, five operations instead of eight, costs registers
// and its second copy of the pass more than it saves (270 us).
__device__ __forceinline__ f32x2 tanh_pair(f32x2 x) {
  const f32x2 y = f2_mul(x, x);
  f32x2 q = f2_fma(f2_pack(-2.983081579e-03f, -2.983081579e-03f), y, f2_pack(1.653281572e-02f, 1.653281572e-02f));
  q = f2_fma(q, y, f2_pack(-5.142535359e-02f, -5.142535359e-02f));
  q = f2_fma(q, y, f2_pack(1.327561524e-01f, 1.327561524e-01f));
  q = f2_fma(q, y, f2_pack(-3.332866991e-01f, -3.332866991e-01f));
  return f2_fma(f2_mul(q, y), x, x);
}

// bf16 A and B, f32 accumulate, M = 128, N = n; B either K-major (0) or MN-major (1).
__host__ __device__ constexpr uint32_t idesc(uint32_t n, uint32_t b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn_major << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void tma_4d(uint32_t dst, const void* tm, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
               ::"r"(dst), "l"(tm), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const void* tm, int c0, int c1, int c2, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               ::"r"(dst), "l"(tm), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}

template <int D, bool FP4>
struct PromptShape {
  static constexpr int HALVES = D / 64;
  static constexpr int TILE = HALVES * HALF;                     // a K or V tile
  static constexpr int Q_BYTES = 2 * HALVES * QT * 128;
  static constexpr int SMEM = (KSTAGES + VSTAGES) * TILE + Q_BYTES + 1024 + 512;
  static constexpr int THREADS = FP4 ? 512 : 384;
  static constexpr int LOADERS = FP4 ? 4 : 1;                    // arrivals on a full barrier
};

// Where a block of query tokens lies: the y-th block of the batch (one warp).
struct BlockPlace { uint32_t b; int token0, first, count; };   // first: of the sequence's tokens; count 0: no such block
__device__ __forceinline__ BlockPlace find_block(const PromptParams& p, uint32_t y, uint32_t lane) {
  BlockPlace at{0, 0, 0, 0};
  const uint32_t step = 2 * p.tile_tokens;
  uint32_t base = 0;
  for (uint32_t i0 = 0; i0 < p.c.batch; i0 += 32) {
    const uint32_t i = i0 + lane;
    int t0 = 0, n = 0;
    if (i < p.c.batch) {
      t0 = __ldg(p.cu_q + i);
      n = __ldg(p.cu_q + i + 1) - t0;
      // a list that does not ascend within the tokens has no blocks where it is wrong
      if (t0 < 0 || n < 0 || uint32_t(t0) + uint32_t(n) > p.tokens) n = 0;
    }
    const uint32_t mine = (uint32_t(n) + step - 1) / step;
    uint32_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= uint32_t(o)) inc += up;
    }
    const uint32_t hit = __ballot_sync(0xFFFFFFFFu, base + inc > y);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const uint32_t nth = y - base - __shfl_sync(0xFFFFFFFFu, inc - mine, src);   // from the sequence's last block down
      const uint32_t all = __shfl_sync(0xFFFFFFFFu, mine, src);
      const int nn = __shfl_sync(0xFFFFFFFFu, n, src);
      at.b = i0 + src;
      at.token0 = __shfl_sync(0xFFFFFFFFu, t0, src);
      at.first = int((all - 1 - nth) * step);
      at.count = min(int(step), nn - at.first);
      return at;
    }
    base += __shfl_sync(0xFFFFFFFFu, inc, 31);
  }
  return at;
}

template <int D, bool FP4, bool CAPPED, bool BIASED>
__global__ void __launch_bounds__(PromptShape<D, FP4>::THREADS, 1)
paged_prompt_kernel(const __grid_constant__ PromptParams p) {
  using Shape = PromptShape<D, FP4>;
  constexpr int HALVES = Shape::HALVES, TILE = Shape::TILE;
  constexpr uint32_t S_COL = 0, O_COL = 256, TMEM_COLS = 512;       // S_t at 128 t, O_t at 256 + D t
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t k_smem = base, v_smem = base + KSTAGES * TILE, q_smem = v_smem + VSTAGES * TILE;
  const uint32_t bar_base = q_smem + Shape::Q_BYTES;
  auto k_full = [&](int s) { return bar_base + 8u * s; };
  auto k_empty = [&](int s) { return bar_base + 8u * (2 + s); };
  auto v_full = [&](int s) { return bar_base + 8u * (4 + s); };
  auto v_empty = [&](int s) { return bar_base + 8u * (6 + s); };
  const uint32_t q_full = bar_base + 8u * 8, tail_bar = bar_base + 8u * 9, drain_bar = bar_base + 8u * 10;
  auto s_full = [&](int t) { return bar_base + 8u * (11 + t); };
  auto p_full = [&](int t, int u) { return bar_base + 8u * (13 + 2 * t + u); };
  auto pva_done = [&](int t) { return bar_base + 8u * (17 + t); };
  auto o_done = [&](int t) { return bar_base + 8u * (19 + t); };
  uint32_t* tmem_ptr_smem = reinterpret_cast<uint32_t*>(gen + (bar_base - base) + 8 * 22);
  volatile int* abort_smem = reinterpret_cast<volatile int*>(tmem_ptr_smem + 1);
  int* place = reinterpret_cast<int*>(tmem_ptr_smem + 2);           // b, token0, first, count
  int* tflag = p.flags ? p.flags + MB_FLAG_WAIT_TIMEOUT : nullptr;

  const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x >> 5), 0);
  const uint32_t lane = threadIdx.x & 31;
  const uint32_t kvh = blockIdx.x % p.c.kv_heads, y = blockIdx.x / p.c.kv_heads, split = blockIdx.y;

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(k_full(s), Shape::LOADERS);
      mbar_init(k_empty(s), 1);
      mbar_init(v_full(s), Shape::LOADERS);
      mbar_init(v_empty(s), 1);
    }
    mbar_init(q_full, 1);
    mbar_init(tail_bar, 1);
    mbar_init(drain_bar, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full(t), 1);
      mbar_init(p_full(t, 0), 128);
      mbar_init(p_full(t, 1), 128);
      mbar_init(pva_done(t), 1);
      mbar_init(o_done(t), 1);
    }
    *abort_smem = 0;
    fence_barrier_init();
    tma_prefetch_desc(&p.tmap_q);
    if (!FP4) {
      tma_prefetch_desc(&p.tmap_k);
      tma_prefetch_desc(&p.tmap_v);
    }
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_ptr_smem), TMEM_COLS);
    tmem_relinquish();
  }
  mb_grid_dependency_sync();
  if (warp == 0) {
    const BlockPlace at = find_block(p, y, lane);
    if (lane == 0) {
      place[0] = int(at.b); place[1] = at.token0; place[2] = at.first; place[3] = at.count;
      if (p.splits > 1 && kvh == 0 && split == 0) p.meta[y] = make_int4(at.token0 + at.first, at.count, 0, 0);
      if (at.count > 0 && paged_len_bad(p.c, at.b)) paged_raise(p.c, at.b);
    }
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem_base = *tmem_ptr_smem;
  const uint32_t b = uint32_t(place[0]);
  const int count = place[3];                                       // tokens of this block
  const int token0 = place[1] + place[2];
  int len = 0, q_first = 0;
  PagedSpan span{};
  if (count > 0) {
    len = paged_len(p.c, b);
    const int n_seq = __ldg(p.cu_q + b + 1) - place[1];
    q_first = len - n_seq + place[2];                               // position of the block's first token
    span = paged_span(p.c, b, len, q_first, q_first + count - 1, BC);
  }
  // this CTA's part of the block's tiles
  const uint32_t all_tiles = span.count();
  const uint32_t per = p.splits > 1 ? max(MIN_SPLIT_TILES, (all_tiles + p.splits - 1) / p.splits) : all_tiles;
  const uint32_t i_first = min(all_tiles, split * per);
  const uint32_t n_tiles = min(per, all_tiles - i_first);
  const int tile_tokens = int(p.tile_tokens);

  const bool loader = warp == 0 || warp >= 12;
  if (loader && n_tiles > 0) {
    if (warp == 0) {
      if (elect_one()) {
        const uint32_t half_bytes = p.tile_tokens * p.group * 128u;
        mbar_arrive_expect_tx(q_full, 2u * HALVES * half_bytes);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int hf = 0; hf < HALVES; ++hf)
            tma_3d(q_smem + (t * HALVES + hf) * (QT * 128), &p.tmap_q, hf * 64, int(kvh * p.group), token0 + t * tile_tokens, q_full);
      }
      __syncwarp();
    }
    if (FP4 && warp == 0) {
      // the queries are all it loads
    } else if (!FP4) {
      // ------------------------------ producer: tiles by TMA ------------------------------
      const uint32_t per_tile = BC / p.box_rows;
      auto pages_of = [&](uint32_t box) -> uint32_t {
        const uint32_t i = box / per_tile;
        if (i >= n_tiles) return p.c.pages;
        const uint32_t r = span.tile_down(i_first + i) * BC + (box % per_tile) * p.box_rows;
        if (!span.needed(int(r), int(p.box_rows))) return p.c.pages;        // zeros
        return paged_page(p.c, b, mb_fastdiv_q(r, p.c.page_div));
      };
      // pages of the next 32 boxes, a lane each, fetched a window ahead; V runs a tile behind K
      uint32_t ids = pages_of(lane), ids_next = pages_of(lane + 32), ids_last = ids;
      auto load_tile = [&](const CUtensorMap* tm, uint32_t dst, uint32_t i, uint32_t from, uint32_t bar) {
        if (elect_one()) mbar_arrive_expect_tx(bar, TILE);
        __syncwarp();
        const uint32_t row0 = span.tile_down(i_first + i) * BC;
        for (uint32_t x = 0; x < per_tile; ++x) {
          const uint32_t page = __shfl_sync(0xFFFFFFFFu, from, (i * per_tile + x) & 31u);
          const uint32_t r = row0 + x * p.box_rows, in_page = r - mb_fastdiv_q(r, p.c.page_div) * p.c.page_size;
          if (elect_one()) {
#pragma unroll
            for (int hf = 0; hf < HALVES; ++hf)
              tma_4d(dst + hf * HALF + x * p.box_rows * 128u, tm, hf * 64, int(kvh), int(in_page), int(page), bar);
          }
          __syncwarp();
        }
      };
      bool ok = true;
      uint32_t tails = 0;
      for (uint32_t i = 0; ok && i <= n_tiles; ++i) {
        if (i > 0) ids_last = ids;                                // the window tile i - 1 was read with
        if (i < n_tiles) {
          if (i > 0 && ((i * per_tile) & 31u) == 0) {
            ids = ids_next;
            ids_next = pages_of(i * per_tile + 32 + lane);
          }
          const int st = int(i % KSTAGES);
          if (!mbar_wait(k_empty(st), ((i / KSTAGES) & 1u) ^ 1u, abort_smem, tflag, 31)) { ok = false; break; }
          load_tile(&p.tmap_k, k_smem + st * TILE, i, ids, k_full(st));
        }
        if (i > 0) {
          const uint32_t j = i - 1;
          const int st = int(j % VSTAGES);
          if (!mbar_wait(v_empty(st), ((j / VSTAGES) & 1u) ^ 1u, abort_smem, tflag, 30)) { ok = false; break; }
          const uint32_t row0 = span.tile_down(i_first + j) * BC, dst = v_smem + st * TILE;
          if (int(row0 + BC) <= len) {
            load_tile(&p.tmap_v, dst, j, ids_last, v_full(st));
          } else {
            // rows behind the length may hold anything, NaN included, and 0 * NaN is NaN: they become zeros before the
            // products may read the tile
            load_tile(&p.tmap_v, dst, j, ids_last, tail_bar);
            if (!mbar_wait(tail_bar, tails & 1u, abort_smem, tflag, 29)) { ok = false; break; }
            ++tails;
            const uint32_t r0 = uint32_t(max(len - int(row0), 0));
            for (uint32_t x = lane; x < (BC - r0) * 8u * HALVES; x += 32) {
              const uint32_t hf = x / ((BC - r0) * 8u), in = x % ((BC - r0) * 8u);
              *reinterpret_cast<uint4*>(gen + (dst - base) + hf * HALF + (r0 + (in >> 3)) * 128u + (in & 7u) * 16u) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(v_full(st));
          }
        }
      }
    } else {
      // ------------------------------ expanders: rows 32 e .. 32 e + 31 of a tile ------------------------------
      // A lane takes 16 bytes of codes (32 features, two scales) of a row: D / 32 lanes to a row.
      const uint32_t e = uint32_t(warp) - 12u;
      constexpr int PER = D / 32, CH = PER;                     // lanes per row; 16-byte loads per lane and tile
      const uint32_t q = lane % PER, row_in = lane / PER;       // rows row_in + i * (32 / PER)
      uint4 codes[CH], codes_next[CH];
      uint32_t sc[CH], sc_next[CH];
      // pages of the warp's two 16-row groups of the next 16 tiles, a lane each, fetched a window ahead
      auto pages_of = [&](uint32_t x) -> uint32_t {
        const uint32_t i = x >> 1;
        if (i >= n_tiles) return p.c.pages;
        const uint32_t r = span.tile_down(i_first + i) * BC + e * 32u + (x & 1u) * 16u;
        if (!span.needed(int(r), 16)) return p.c.pages;
        return paged_page(p.c, b, mb_fastdiv_q(r, p.c.page_div));
      };
      uint32_t ids = pages_of(lane), ids_next = pages_of(32 + lane);
      // loads of half-step h: K of tile h / 2 for even h, V for odd h; rows that are not there become zeros
      auto fetch = [&](uint32_t h, uint4* cd, uint32_t* s2) {
        const uint32_t i = h >> 1;
        if (i >= n_tiles) return;
        if ((h & 31u) == 0 && h > 0) { ids = ids_next; ids_next = pages_of(h + 32 + lane); }
        const uint8_t* pc = (h & 1u) ? p.v : p.k;
        const uint8_t* ps = (h & 1u) ? p.vs : p.ks;
        const uint32_t r0 = span.tile_down(i_first + i) * BC + e * 32u;
#pragma unroll
        for (int x = 0; x < CH; ++x) {
          const uint32_t in = row_in + x * (32 / PER), r = r0 + in, r16 = r0 + (in & 16u);
          const uint32_t page = __shfl_sync(0xFFFFFFFFu, ids, (h & 30u) + (x * (32 / PER) >= 16 ? 1u : 0u));
          cd[x] = make_uint4(0, 0, 0, 0);
          s2[x] = 0;
          if (int(r) < len && page < p.c.pages) {
            const uint32_t in_page = r16 - mb_fastdiv_q(r16, p.c.page_div) * p.c.page_size + (in & 15u);
            const size_t at = (size_t(page) * p.c.page_size + in_page) * p.c.kv_heads + kvh;
            cd[x] = __ldg(reinterpret_cast<const uint4*>(pc + at * (D / 2)) + q);
            s2[x] = __ldg(reinterpret_cast<const uint16_t*>(ps + at * (D / 16)) + q);
          }
        }
      };
      auto expand = [&](uint32_t dst) {
#pragma unroll
        for (int x = 0; x < CH; ++x) {
          const uint32_t row = e * 32u + row_in + x * (32 / PER);
          uint32_t sh;
          asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(sh) : "h"(uint16_t(sc[x])));
          const float2 sf = __half22float2(*reinterpret_cast<__half2*>(&sh));
          // the f16 pattern of an E2M1 value moved three places is the bf16 pattern of value * 2^-112
          const __nv_bfloat162 s_lo = __float2bfloat162_rn(sf.x * 5.192296858534828e33f), s_hi = __float2bfloat162_rn(sf.y * 5.192296858534828e33f);
          const uint32_t w[4] = {codes[x].x, codes[x].y, codes[x].z, codes[x].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // chunk order rotated by the lane's half of the row, so that eight lanes' stores hit eight bank groups
            const int ii = i ^ (int(q >> 1) << 1);
            const uint32_t ww = ii == 0 ? w[0] : ii == 1 ? w[1] : ii == 2 ? w[2] : w[3];
            uint32_t h[4];
            asm("{ .reg .b8 b0, b1, b2, b3; mov.b32 {b0, b1, b2, b3}, %4;\n\t"
                "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
                "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3; }"
                : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(ww));
            const __nv_bfloat162 s2 = ii < 2 ? s_lo : s_hi;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              uint32_t m = (h[n] & 0x80008000u) | ((h[n] >> 3) & 0x0FFF0FFFu);
              const __nv_bfloat162 r = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&m), s2);
              h[n] = *reinterpret_cast<const uint32_t*>(&r);
            }
            const uint32_t c = q * 4u + uint32_t(ii);
            *reinterpret_cast<uint4*>(gen + (dst - base) + (c >> 3) * HALF + row * 128u + (((c & 7u) ^ (row & 7u)) << 4)) =
                make_uint4(h[0], h[1], h[2], h[3]);
          }
        }
        fence_proxy_async();
        __syncwarp();
      };
      fetch(0, codes, sc);
      for (uint32_t h = 0; h < 2 * n_tiles; ++h) {
        fetch(h + 1, codes_next, sc_next);
        const uint32_t i = h >> 1;
        const int st = int(i & 1u);
        const uint32_t empty = (h & 1u) ? v_empty(st) : k_empty(st);
        if (!mbar_wait(empty, ((i >> 1) & 1u) ^ 1u, abort_smem, tflag, 28)) break;
        expand(((h & 1u) ? v_smem : k_smem) + st * TILE);
        if (lane == 0) mbar_arrive((h & 1u) ? v_full(st) : k_full(st));
#pragma unroll
        for (int x = 0; x < CH; ++x) { codes[x] = codes_next[x]; sc[x] = sc_next[x]; }
      }
    }
  } else if (warp == 1 && n_tiles > 0) {
    // ------------------------------ issuer ------------------------------
    bool ok = mbar_wait(q_full, 0u, abort_smem, tflag, 32);
    const uint32_t id_s = idesc(BC, 0), id_pv = idesc(D, 1);
    auto issue_s = [&](int t, uint32_t j) {
      if (elect_one()) {
        const uint32_t k0 = k_smem + (j % KSTAGES) * TILE;
#pragma unroll
        for (int hf = 0; hf < HALVES; ++hf) {
          const uint64_t adesc = make_kmajor_sw128_desc(q_smem + (t * HALVES + hf) * (QT * 128));
          const uint64_t bdesc = make_kmajor_sw128_desc(k0 + hf * HALF);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_f16(tmem_base + S_COL + 128 * t, adesc + 2 * kk, bdesc + 2 * kk, id_s, (hf | kk) != 0);
        }
        umma_commit(s_full(t));
        if (t == 1) umma_commit(k_empty(int(j % KSTAGES)));
      }
      __syncwarp();
    };
    if (ok) ok = mbar_wait(k_full(0), 0u, abort_smem, tflag, 33);
    if (ok) {
      fence_after_sync();
      issue_s(0, 0);
      issue_s(1, 0);
    }
    for (uint32_t j = 0; ok && j < n_tiles; ++j) {
      const int vst = int(j % VSTAGES);
      for (int t = 0; t < 2 && ok; ++t) {
        for (int u = 0; u < 2; ++u) {
          if (!mbar_wait(p_full(t, u), j & 1u, abort_smem, tflag, 34)) { ok = false; break; }
          if (t == 0 && u == 0 && !mbar_wait(v_full(vst), (j / VSTAGES) & 1u, abort_smem, tflag, 35)) { ok = false; break; }
          fence_after_sync();
          if (elect_one()) {
            const uint32_t a_tmem = tmem_base + S_COL + 128 * t + 64 * u;      // P of 64 keys: 32 columns of bf16 pairs
            // V: MN-major, 64-feature blocks HALF apart, 8-key groups 1 KB apart
            const uint64_t bdesc = make_smem_desc(v_smem + vst * TILE + u * (64 * 128), HALF, 1024, LAYOUT_SWIZZLE_128B);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_f16_ts(tmem_base + O_COL + D * t, a_tmem + 8 * kk, bdesc + 128 * kk, id_pv, (j | uint32_t(u) | uint32_t(kk)) != 0u);
            if (u == 0) umma_commit(pva_done(t));
            else if (t == 1) umma_commit(v_empty(vst));
            if (u == 1 && j + 1 == n_tiles) umma_commit(o_done(t));
          }
          __syncwarp();
        }
        if (!ok) break;
        if (j + 1 < n_tiles) {
          if (t == 0) {
            if (!mbar_wait(k_full(int((j + 1) % KSTAGES)), ((j + 1) / KSTAGES) & 1u, abort_smem, tflag, 33)) { ok = false; break; }
            fence_after_sync();
          }
          issue_s(t, j + 1);
        }
      }
    }
    if (!ok) {
      if (elect_one()) umma_commit(drain_bar);
      __syncwarp();
      long long t0 = clock64();
      while (!mbar_try_wait(drain_bar, 0u) && clock64() - t0 < WAIT_LIMIT_CYCLES) {}
    }
  } else if (warp >= 4 && warp < 12) {
    // ------------------------------ softmax groups: a thread per query row ------------------------------
    const int t = (warp - 4) >> 2;
    const uint32_t quad = uint32_t(warp) & 3u, r = quad * 32u + lane;       // TMEM lanes of this warp, row of the tile
    const uint32_t tok_in = mb_fastdiv_q(r, p.group_div), hg = r - tok_in * p.group;
    const int tok = t * tile_tokens + int(tok_in);                // token of the block
    const bool mine = tok_in < p.tile_tokens && tok < count;      // a row of `out`
    const int qpos = q_first + tok;
    const bool live = mine && qpos >= 0;
    const uint32_t lane_addr = (quad * 32u) << 16;
    const uint32_t t_s = tmem_base + lane_addr + S_COL + 128 * t, t_o = tmem_base + lane_addr + O_COL + D * t;
    const float mult = CAPPED ? p.cap_log2 : p.scale_log2;
    const float slope = BIASED && mine ? __ldg(p.slopes + kvh * p.group + hg) * 1.4426950408889634f : 0.0f;
    const int window = p.c.window ? int(p.c.window) : 0x40000000;
    const bool idle = !__any_sync(0xFFFFFFFFu, live);           // no row of the warp has a query: its P may stay what it is
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (uint32_t j = 0; ok && j < n_tiles; ++j) {
      const int tile0 = int(span.tile_down(i_first + j) * BC);
      if (!mbar_wait(s_full(t), j & 1u, abort_smem, tflag, 37)) { ok = false; break; }
      fence_after_sync();
#pragma unroll 1
      for (int u = 0; u < 2; ++u) {
        const int kabs = tile0 + 64 * u;
        // keys [first, vis) of this unit's 64 are in the row's band, keys below pre in its prefix
        const int vis = live ? min(len, qpos + 1) - kabs : 0;
        const int first = qpos + 1 - window - kabs;
        const int pre = live ? span.prefix - kabs : 0;
        const bool begin = j == 0 && u == 0;
        uint32_t w[32];
        float sum = 0.0f;
        // The ordinary unit: every key seen by every row of the warp (what rows without a query hold does not matter),
        // references at hand.
        bool done = !begin && !idle && __all_sync(0xFFFFFFFFu, !live || (m > -INFINITY && ((vis >= 64 && first <= 0) || (pre >= 64 && (!BIASED || qpos >= kabs + 63)))));
        if (done) {
          uint32_t sr[64];
          tmem_ld_x32(t_s + 64 * u, sr);
          tmem_ld_x32(t_s + 64 * u + 32, sr + 32);
          tmem_ld_wait();
          const f32x2 mult2 = f2_pack(mult, mult);
          if (CAPPED) {
            float big = 0.0f;
#pragma unroll
            for (int i = 0; i < 64; ++i) big = fmaxf(big, fabsf(__uint_as_float(sr[i])));
            // scores beyond the cap are left to the general form (NaN passes here)
            done = __all_sync(0xFFFFFFFFu, big * p.inv_cap <= 1.0f || !live);
            const f32x2 c2 = f2_pack(p.inv_cap, p.inv_cap);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float a0, a1;
              f2_unpack(tanh_pair(f2_mul(f2_pack(__uint_as_float(sr[2 * i]), __uint_as_float(sr[2 * i + 1])), c2)), a0, a1);
              sr[2 * i] = __float_as_uint(a0);
              sr[2 * i + 1] = __float_as_uint(a1);
            }
          }
          // the keys are at or before the query, so the bias is linear in the key
          const float off = BIASED ? fmaf(-slope, float(qpos - kabs), -m) : -m;
          f32x2 off2 = f2_pack(off, off + slope);
          const f32x2 step2 = f2_pack(2.0f * slope, 2.0f * slope);
          f32x2 acc0 = f2_pack(0.0f, 0.0f), acc1 = acc0;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float x0, x1;
            f2_unpack(f2_fma(f2_pack(__uint_as_float(sr[2 * i]), __uint_as_float(sr[2 * i + 1])), mult2, off2), x0, x1);
            x0 = paged_ex2(x0);
            x1 = paged_ex2(x1);
            if (i & 1) acc1 = f2_add(acc1, f2_pack(x0, x1)); else acc0 = f2_add(acc0, f2_pack(x0, x1));
            w[i] = pack2(x0, x1);
            if (BIASED) off2 = f2_add(off2, step2);
          }
          float a0, a1, b0, b1;
          f2_unpack(acc0, a0, a1);
          f2_unpack(acc1, b0, b1);
          sum = (a0 + a1) + (b0 + b1);
          done = done && !__any_sync(0xFFFFFFFFu, live && !(sum <= 1099511627776.0f));
        }
        if (!done && !idle) {
          // The general form: masks, and the move of the references. Scores in units of log2 are taken from tensor memory
          // again, 32 at a time; which of them the row sees is a word of bits.
          auto bits = [&](int h) -> uint32_t {
            auto below = [](int n) -> uint32_t { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; };
            return (below(vis - 32 * h) & ~below(first - 32 * h)) | below(pre - 32 * h);
          };
          auto scores = [&](int h, float* x) {
            uint32_t sr[32];
            tmem_ld_x32(t_s + 64 * u + 32 * h, sr);
            tmem_ld_wait();
            const uint32_t seen = bits(h);
            const float away = float(qpos - kabs - 32 * h);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float y = __uint_as_float(sr[i]);
              y = (CAPPED ? paged_tanh(y * p.inv_cap, true) : y) * mult;
              if (BIASED) y = fmaf(-slope, fabsf(away - float(i)), y);
              x[i] = seen & (1u << i) ? y : -INFINITY;
            }
          };
          // a row that sees its first keys needs a reference
          bool move = __any_sync(0xFFFFFFFFu, m == -INFINITY && (bits(0) | bits(1)) != 0u);
          for (;;) {
            if (move) {
              float mx = -INFINITY;
#pragma unroll 1
              for (int h = 0; h < 2; ++h) {
                float x[32];
                scores(h, x);
#pragma unroll
                for (int i = 0; i < 32; ++i) mx = fmaxf(mx, x[i]);
              }
              // the other rows' references move where they are 2^20 and more behind
              const float m_new = mx > m + 20.0f ? mx : m;
              if (!begin && __any_sync(0xFFFFFFFFu, m_new != m)) {
                // O must be at rest: the products of the unit before this one are done once S(j) is (u = 0) or once
                // pva_done says so (u = 1)
                const float f = m == -INFINITY ? 0.0f : paged_ex2(m - m_new);
                if (u == 1 && !mbar_wait(pva_done(t), j & 1u, abort_smem, tflag, 38)) { ok = false; break; }
                fence_after_sync();
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                  uint32_t v[32];
                  tmem_ld_x32(t_o + c * 32, v);
                  tmem_ld_wait();
#pragma unroll
                  for (int i = 0; i < 32; ++i) v[i] = m_new == m ? v[i] : __float_as_uint(__uint_as_float(v[i]) * f);
                  tmem_st_x32(t_o + c * 32, v);
                }
                tmem_st_wait();
                if (m_new != m) l *= f;
              }
              m = m_new;
            }
            const float off = m == -INFINITY ? 0.0f : m;
            sum = 0.0f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float x[32];
              scores(h, x);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float p0 = paged_ex2(x[2 * i] - off), p1 = paged_ex2(x[2 * i + 1] - off);
                sum += p0 + p1;
                w[16 * h + i] = pack2(p0, p1);
              }
            }
            if (move) break;
            move = __any_sync(0xFFFFFFFFu, live && !(sum <= 1099511627776.0f));
            if (!move) break;
          }
          if (!ok) break;
        }
        if (!idle) {
          tmem_st_x32(t_s + 64 * u, w);
          tmem_st_wait();
          l += sum;
        }
        fence_before_sync();
        mbar_arrive(p_full(t, u));
      }
    }
    if (ok && n_tiles > 0) ok = mbar_wait(o_done(t), 0u, abort_smem, tflag, 40);
    fence_after_sync();
    if (!live) l = 0.0f;
    if (p.splits == 1) {
      const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
      __nv_bfloat16* dst_row = p.out + (size_t(token0 + tok) * p.heads + kvh * p.group + hg) * D;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t v[32];
        if (n_tiles > 0) {
          tmem_ld_x32(t_o + c * 32, v);
          tmem_ld_wait();
        }
        if (mine && ok) {
          uint4* dst = reinterpret_cast<uint4*>(dst_row + c * 32);
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            uint32_t o4[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              o4[i] = l == 0.0f ? 0u : pack2(__uint_as_float(v[8 * g + 2 * i]) * inv, __uint_as_float(v[8 * g + 2 * i + 1]) * inv);
            dst[g] = make_uint4(o4[0], o4[1], o4[2], o4[3]);
          }
        }
      }
    } else if (count > 0) {
      float* dst = p.part + (((size_t(y) * p.c.kv_heads + kvh) * p.splits + split) * (2 * QT) + t * QT + r) * (D + 4);
      if (mine && ok) {
        dst[D] = m;
        dst[D + 1] = l;
      }
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t v[32];
        if (n_tiles > 0) {
          tmem_ld_x32(t_o + c * 32, v);
          tmem_ld_wait();
        }
        if (mine && ok && l != 0.0f) {
#pragma unroll
          for (int g = 0; g < 8; ++g)
            *reinterpret_cast<uint4*>(dst + c * 32 + 4 * g) = make_uint4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
        }
      }
    }
  }

  fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    fence_after_sync();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// Joins the key parts of a block: a warp per (token, head) row, four values (two at D = 64) per lane, parts in order.
template <int D>
__global__ void __launch_bounds__(256)
paged_prompt_join_kernel(const __grid_constant__ PromptParams p) {
  constexpr int V = D / 32;
  mb_grid_dependency_sync();
  const uint32_t kvh = blockIdx.x % p.c.kv_heads, y = blockIdx.x / p.c.kv_heads, lane = threadIdx.x & 31;
  const int4 meta = p.meta[y];
  for (uint32_t r = blockIdx.y * 8 + (threadIdx.x >> 5); r < 2 * QT; r += 8 * gridDim.y) {
    const uint32_t t = r / QT, in = r % QT, tok_in = mb_fastdiv_q(in, p.group_div), hg = in - tok_in * p.group;
    const int tok = int(t * p.tile_tokens + tok_in);
    if (tok_in >= p.tile_tokens || tok >= meta.y) continue;
    const float* src = p.part + ((size_t(y) * p.c.kv_heads + kvh) * p.splits * (2 * QT) + r) * (D + 4);
    const size_t step = size_t(2 * QT) * (D + 4);
    float mm = -INFINITY, ll = 0.0f, acc[V] = {};
    for (uint32_t s = 0; s < p.splits; ++s) mm = fmaxf(mm, src[s * step + D]);
    for (uint32_t s = 0; s < p.splits; ++s) {
      const float ls = src[s * step + D + 1];
      if (ls == 0.0f) continue;                    // its values were not written
      const float f = exp2f(src[s * step + D] - mm);
      ll = fmaf(ls, f, ll);
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = fmaf(src[s * step + lane * V + i], f, acc[i]);
    }
    const float inv = ll > 0.0f ? 1.0f / ll : (ll == 0.0f ? 0.0f : ll);
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + (size_t(meta.x + tok) * p.heads + kvh * p.group + hg) * D) + lane * (V / 2);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) dst[i] = pack2(acc[2 * i] * inv, acc[2 * i + 1] * inv);
  }
}

template <int D, bool FP4, bool CAPPED, bool BIASED>
int launch_prompt(mb_ctx* ctx, cudaStream_t stream, const PromptParams& p) {
  using Shape = PromptShape<D, FP4>;
  constexpr uint32_t once_bit = 1u << (8 + (D == 128) + 2 * FP4 + 4 * CAPPED + 8 * BIASED);
  if (!(ctx->paged_once.load(std::memory_order_acquire) & once_bit)) {
    MB_CUDA_OK(ctx, cudaFuncSetAttribute(paged_prompt_kernel<D, FP4, CAPPED, BIASED>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::SMEM));
    ctx->paged_once.fetch_or(once_bit, std::memory_order_release);
  }
  MB_CUDA_OK(ctx, mb_launch_pdl(paged_prompt_kernel<D, FP4, CAPPED, BIASED>, dim3(p.blocks * p.c.kv_heads, p.splits), dim3(Shape::THREADS),
                                Shape::SMEM, stream, p));
  if (p.splits > 1)
    MB_CUDA_OK(ctx, mb_launch_pdl(paged_prompt_join_kernel<D>, dim3(p.blocks * p.c.kv_heads, 8), dim3(256), 0, stream, p));
  return MB_OK;
}

struct PromptPlan { uint32_t tile_tokens, blocks, splits; size_t meta_bytes, bytes; };
PromptPlan prompt_plan(const mb_ctx* ctx, const mb_paged_kv* kv, size_t tokens, size_t heads) {
  PromptPlan r{};
  const size_t group = heads / kv->kv_heads;
  r.tile_tokens = uint32_t(QT / group);
  // no batch cuts into more blocks than this; those past the real ones end at once
  r.blocks = uint32_t(tokens / (2 * r.tile_tokens) + std::min(kv->batch, tokens));
  // Key parts of a block: as many as there are SMs for, of at least four tiles each (32 / 8 heads of 128, one part / two /
  // four / eight / what this gives: 232 / 132 / 79 / 60 / 60 us for 64 tokens over 16000 rows, 41 / 37 / 32 / 35 / 32 over
  // 2000, 238 / 136 / 149 / 143 / 103 for 300 tokens over 16000: more parts than SMs wait for a second wave).
  const size_t ctas = size_t(r.blocks) * kv->kv_heads, longest = kv->table_width * kv->page_size;
  size_t s = size_t(ctx->sm_count) / std::max<size_t>(1, ctas);
  s = std::min<size_t>(std::min<size_t>(s, MAX_SPLITS), longest / (BC * MIN_SPLIT_TILES));
  r.splits = uint32_t(std::max<size_t>(1, s));
  if (r.splits > 1) {
    r.meta_bytes = (r.blocks * sizeof(int4) + 255) / 256 * 256;
    r.bytes = r.meta_bytes + ctas * r.splits * 2 * QT * (kv->d + 4) * sizeof(float);
  }
  return r;
}

}  // namespace

MB_API size_t mb_paged_prompt_workspace(mb_ctx* ctx, const mb_paged_kv* kv, size_t tokens, size_t heads) {
  if (!ctx || !kv || tokens == 0 || kv->kv_heads == 0 || heads == 0 || heads % kv->kv_heads != 0 || heads / kv->kv_heads > QT ||
      kv->batch == 0)
    return 0;
  return prompt_plan(ctx, kv, tokens, heads).bytes;
}

MB_API int mb_paged_prompt(mb_ctx* ctx, mb_stream stream_, const void* q, size_t tokens, size_t heads, const mb_paged_kv* kv,
                           const int32_t* cu_q, const mb_score_terms* terms, void* out, void* workspace, size_t workspace_bytes) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  PromptParams p;
  MB_REQUIRE(ctx, ctx && terms, "paged_prompt: null argument");
  int rc = paged_view(ctx, "paged_prompt", kv, terms, heads, &p.c);
  if (rc) return rc;
  MB_REQUIRE(ctx, cu_q && (tokens == 0 || (q && out)) && mb_aligned(cu_q, 4) && mb_aligned(q, 16) && mb_aligned(out, 16),
             "paged_prompt: null argument, or q and out without 16-byte alignment");
  MB_REQUIRE(ctx, heads / kv->kv_heads <= QT, "paged_prompt: at most %d query heads per KV head, got %zu", QT, heads / kv->kv_heads);
  if (tokens == 0) return MB_OK;
  const PromptPlan plan = prompt_plan(ctx, kv, tokens, heads);
  MB_REQUIRE(ctx, tokens < (1ull << 30) && size_t(plan.blocks) * kv->kv_heads < (1ull << 31), "paged_prompt: too many tokens");
  MB_REQUIRE(ctx, plan.bytes == 0 || (workspace && workspace_bytes >= plan.bytes && mb_aligned(workspace, 256)),
             "paged_prompt: needs %zu workspace bytes, 256-byte aligned", plan.bytes);
  const bool fp4 = kv->elem == MB_KV_NVFP4;
  p.k = static_cast<const uint8_t*>(kv->k); p.v = static_cast<const uint8_t*>(kv->v);
  p.ks = static_cast<const uint8_t*>(kv->k_scales); p.vs = static_cast<const uint8_t*>(kv->v_scales);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.cu_q = cu_q;
  p.slopes = terms->slopes;
  p.meta = static_cast<int4*>(workspace);
  p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.meta_bytes);
  p.tokens = uint32_t(tokens); p.heads = uint32_t(heads); p.group = uint32_t(heads / kv->kv_heads);
  p.tile_tokens = plan.tile_tokens; p.blocks = plan.blocks; p.splits = plan.splits;
  p.group_div = mb_fastdiv_make(p.group);
  p.scale_log2 = terms->scale * 1.4426950408889634f;
  p.cap_log2 = terms->softcap * 1.4426950408889634f;
  p.inv_cap = terms->softcap > 0.0f ? terms->scale / terms->softcap : 0.0f;
  p.flags = ctx->flags_dev;
  p.box_rows = paged_box_rows(kv->page_size, BC);
  const uint64_t qd[3] = {kv->d, heads, tokens}, qs[2] = {uint64_t(kv->d) * 2, uint64_t(heads) * kv->d * 2};
  const uint32_t qb[3] = {64, p.group, p.tile_tokens};
  rc = paged_encode_map(ctx, &p.tmap_q, 3, q, qd, qs, qb);
  if (rc) return rc;
  if (!fp4) {
    rc = paged_pool_map(ctx, &p.tmap_k, kv->k, kv, p.box_rows);
    if (rc) return rc;
    rc = paged_pool_map(ctx, &p.tmap_v, kv->v, kv, p.box_rows);
    if (rc) return rc;
  } else {
    memset(&p.tmap_k, 0, sizeof p.tmap_k);
    memset(&p.tmap_v, 0, sizeof p.tmap_v);
  }
  const bool cap = terms->softcap > 0.0f, bias = terms->slopes != nullptr;
#define MB_PROMPT(DD, F) \
  rc = cap ? (bias ? launch_prompt<DD, F, true, true>(ctx, stream, p) : launch_prompt<DD, F, true, false>(ctx, stream, p)) \
           : (bias ? launch_prompt<DD, F, false, true>(ctx, stream, p) : launch_prompt<DD, F, false, false>(ctx, stream, p))
  if (kv->d == 128) { if (fp4) MB_PROMPT(128, true); else MB_PROMPT(128, false); }
  else { if (fp4) MB_PROMPT(64, true); else MB_PROMPT(64, false); }
#undef MB_PROMPT
  if (rc) return rc;
  MB_LAUNCH_OK(ctx);
  return MB_OK;
}

// The paged cache: argument checks shared by its kernels, and rotation + append.
//
// Append. One block takes TB tokens: it finds their sequences and rows, takes the d / 2 sines and cosines of each
// token once for all of its heads, and then walks the (token, head) units, d / 16 threads to a unit, a thread holding
// the eight pairs (f, f + d / 2) of two 16-byte loads. Bound by HBM at prompt sizes (each value read once, written
// once) and by the chain cu_q -> length -> table entry -> store at decode sizes; the loads of a thread's first unit
// are issued before that chain. Measured (32 query and 8 KV heads of 128): 3.0 us for one token, 3.4 us for 64, 37.9 us
// for 8192 into bf16 pages (218 MB read and written, 0.88 of the copy rate), 21.4 us for 5095 into NVFP4 pages (110 MB,
// 0.79; there the quantizer's instructions).
#include "paged.cuh"
#include "quant_block.cuh"

namespace {

struct AppendParams {
  PagedView c;
  const uint4* qkv;
  uint4* q_out;
  void *k, *v, *ks, *vs;
  const int32_t* cu_q;
  const int32_t* positions;
  const float* inv_freq;
  uint32_t tokens, per_seq, hq, heads;   // heads = hq + 2 kv_heads
  size_t stride16;                       // row stride of qkv in 16-byte units
  uint32_t axes;
  uint32_t section_end[4];
};

__device__ __forceinline__ void unpack8(uint4 v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ uint4 pack8(const float* f) {
  return make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7]));
}

// Eight of a block's 16 values; the lane beside it (lane ^ 1) holds the others. The arithmetic of quant_block_recip.
__device__ __forceinline__ uint32_t quant_half_recip(uint4 bits, uint32_t& sbyte) {
  float x[8];
  unpack8(bits, x);
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[i]));
  amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
  sbyte = mb_e4m3_encode(fminf(mb_div6(amax), 448.0f));
  const float s = mb_e4m3_decode(sbyte);
  float y[8];
  mb_mul8(x, s > 0.0f ? __frcp_rn(s) : 0.0f, y);
  return mb_cvt_e2m1x8(y);
}

constexpr int APPEND_THREADS = 256;

// G = threads of a unit = d / 16
template <bool FP4, int TB, int G>
__global__ void __launch_bounds__(APPEND_THREADS)
paged_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int HALF = 8 * G;                        // d / 2
  constexpr int UNITS = APPEND_THREADS / G;          // units of a pass
  // (cos, sin) of frequencies 2 i and 2 i + 1 of thread g's eight at [i][g]: the threads of a unit read 16 bytes each, side
  // by side
  __shared__ float4 turn[TB][4][G];
  __shared__ long long slot[TB];                     // pool row of a token; -1: nowhere to go, -2: not a token
  __shared__ int row_of[TB];
  mb_grid_dependency_sync();
  const uint32_t tok0 = blockIdx.x * TB;
  const uint32_t g = threadIdx.x % G;
  const uint32_t units = TB * p.heads;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  auto load = [&](uint32_t u, uint4& lo, uint4& hi) {
    const uint32_t tok = tok0 + u / p.heads;
    if (u < units && tok < p.tokens) {
      const uint4* src = p.qkv + size_t(tok) * p.stride16 + (u % p.heads) * (2 * G);
      lo = __ldg(src + g);
      hi = __ldg(src + G + g);
    }
  };
  uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
  load(threadIdx.x / G + blockIdx.y * UNITS, lo, hi);

  if (warp < TB) {
    // the token's sequence: how many sequences end at or before it
    const uint32_t tok = tok0 + warp;
    uint32_t b = 0;
    int first = 0, n = int(p.per_seq);
    bool live = tok < p.tokens;
    if (p.cu_q) {
      for (uint32_t i0 = 0; i0 < p.c.batch; i0 += 32) {
        const bool done = i0 + lane < p.c.batch && uint32_t(__ldg(p.cu_q + 1 + i0 + lane)) <= tok;
        b += __popc(__ballot_sync(0xFFFFFFFFu, done));
      }
      live = live && b < p.c.batch;
      if (live) {
        first = __ldg(p.cu_q + b);
        n = __ldg(p.cu_q + b + 1) - first;
      }
    } else {
      b = tok / p.per_seq;
      first = int(b * p.per_seq);
      live = live && b < p.c.batch;
    }
    if (lane == 0) {
      long long at = -2;
      int row = 0;
      if (live) {
        const int len = paged_len(p.c, b);
        row = len - n + (int(tok) - first);
        at = -1;
        if (paged_len_bad(p.c, b) || row < 0) paged_raise(p.c, b);
        if (row >= 0 && row < len) {
          const uint32_t e = mb_fastdiv_q(uint32_t(row), p.c.page_div);
          const uint32_t page = paged_page(p.c, b, e);
          if (page < p.c.pages) at = (long long)page * p.c.page_size + (uint32_t(row) - e * p.c.page_size);
        }
      }
      slot[warp] = at;
      row_of[warp] = row;
    }
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < TB * HALF; i += APPEND_THREADS) {
    const uint32_t t = i / HALF, f = i % HALF, tok = tok0 + t;
    if (slot[t] == -2) continue;
    int pos = row_of[t];
    if (p.positions) {
      uint32_t a = 0;
      while (a + 1 < p.axes && f >= p.section_end[a]) ++a;
      pos = __ldg(p.positions + size_t(a) * p.tokens + tok);
    }
    // The angle needs 31 + 24 bits before its multiples of 2 pi are gone; what is left takes 32.
    const double angle = double(pos) * double(__ldg(p.inv_freq + f));
    const double turns = rint(angle * 0.15915494309189535);
    const double rest = fma(-turns, 6.283185307179586, angle);
    const float high = float(rest), low = float(rest - double(high));      // low: what f32 rounds off, up to 2^-23
    float s, c;
    sincosf(high, &s, &c);
    const float s0 = s;
    s = fmaf(low, c, s);
    c = fmaf(-low, s0, c);
    reinterpret_cast<float2*>(&turn[t][(f % 8) / 2][f / 8])[f % 2] = make_float2(c, s);
  }
  __syncthreads();

  const uint32_t kvh = p.c.kv_heads;
  // every lane walks every pass: the quantizer's lanes exchange maxima
  for (uint32_t u0 = blockIdx.y * UNITS; u0 < units; u0 += UNITS * gridDim.y) {
    const uint32_t u = u0 + threadIdx.x / G;
    const uint32_t t = min(u / p.heads, uint32_t(TB - 1)), head = u % p.heads, tok = tok0 + t;
    const uint4 a = lo, b = hi;
    load(u + UNITS * gridDim.y, lo, hi);
    const long long at = u < units ? slot[t] : -2;
    uint4 r0 = a, r1 = b;
    if (head < p.hq + kvh && at != -2) {
      float x[8], y[8], o[8], w[8];
      unpack8(a, x);
      unpack8(b, y);
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float4 cs = turn[t][j / 2][g];
        o[j] = x[j] * cs.x - y[j] * cs.y;
        w[j] = y[j] * cs.x + x[j] * cs.y;
        o[j + 1] = x[j + 1] * cs.z - y[j + 1] * cs.w;
        w[j + 1] = y[j + 1] * cs.z + x[j + 1] * cs.w;
      }
      r0 = pack8(o);
      r1 = pack8(w);
    }
    if (head < p.hq) {
      if (at != -2) {
        uint4* dst = p.q_out + (size_t(tok) * p.hq + head) * (2 * G);
        dst[g] = r0;
        dst[G + g] = r1;
      }
    }
    const bool is_k = head < p.hq + kvh;
    const uint32_t h = is_k ? head - p.hq : head - p.hq - kvh;
    if (!FP4) {
      if (head >= p.hq && at >= 0) {
        uint4* dst = static_cast<uint4*>(is_k ? p.k : p.v) + (size_t(at) * kvh + h) * (2 * G);
        dst[g] = r0;
        dst[G + g] = r1;
      }
    } else if (__any_sync(0xFFFFFFFFu, head >= p.hq)) {      // query heads have nothing to quantize
      uint32_t s0, s1;
      const uint32_t c0 = quant_half_recip(r0, s0), c1 = quant_half_recip(r1, s1);
      if (head >= p.hq && at >= 0) {
        const size_t row = size_t(at) * kvh + h;
        uint32_t* codes = static_cast<uint32_t*>(is_k ? p.k : p.v) + row * (2 * G);
        codes[g] = c0;
        codes[G + g] = c1;
        if ((g & 1u) == 0) {
          uint8_t* sc = static_cast<uint8_t*>(is_k ? p.ks : p.vs) + row * G;
          sc[g / 2] = uint8_t(s0);
          sc[G / 2 + g / 2] = uint8_t(s1);
        }
      }
    }
  }
}

template <bool FP4, int TB>
cudaError_t launch_append(const AppendParams& p, uint32_t d, dim3 grid, cudaStream_t stream) {
  return d == 128 ? mb_launch_pdl(paged_append_kernel<FP4, TB, 8>, grid, dim3(APPEND_THREADS), 0, stream, p)
                  : mb_launch_pdl(paged_append_kernel<FP4, TB, 4>, grid, dim3(APPEND_THREADS), 0, stream, p);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

}  // namespace

int paged_encode_map(mb_ctx* ctx, CUtensorMap* tm, uint32_t rank, const void* base, const uint64_t* dims,
                     const uint64_t* strides_bytes, const uint32_t* box) {
  if (!ctx->encode_tiled) {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult q;
    MB_CUDA_OK(ctx, cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q));
    if (!sym || q != cudaDriverEntryPointSuccess)
      return mb_fail(ctx, MB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    ctx->encode_tiled = sym;
  }
  cuuint64_t cdims[5], cstr[4];
  cuuint32_t cbox[5], estr[5] = {1, 1, 1, 1, 1};
  for (uint32_t i = 0; i < rank; ++i) { cdims[i] = dims[i]; cbox[i] = box[i]; }
  for (uint32_t i = 0; i + 1 < rank; ++i) cstr[i] = strides_bytes[i];
  CUresult r = reinterpret_cast<EncodeTiledFn>(ctx->encode_tiled)(
      tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), cdims, cstr, cbox, estr,
      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return mb_fail(ctx, MB_ERR_CUDA, "cuTensorMapEncodeTiled (paged) failed with %d", int(r));
  return MB_OK;
}

int paged_pool_map(mb_ctx* ctx, CUtensorMap* tm, const void* pool, const mb_paged_kv* kv, uint32_t box_rows) {
  const uint64_t row = uint64_t(kv->kv_heads) * kv->d * 2;
  const uint64_t dims[4] = {kv->d, kv->kv_heads, kv->page_size, kv->pages};
  const uint64_t strides[3] = {uint64_t(kv->d) * 2, row, row * kv->page_size};
  const uint32_t box[4] = {64, 1, box_rows, 1};
  return paged_encode_map(ctx, tm, 4, pool, dims, strides, box);
}

int paged_view(mb_ctx* ctx, const char* what, const mb_paged_kv* kv, const mb_score_terms* terms, size_t heads, PagedView* out) {
  MB_REQUIRE(ctx, ctx != nullptr, "%s: null context", what);
  MB_REQUIRE(ctx, kv && kv->k && kv->v && kv->block_table && kv->lens, "%s: null argument", what);
  MB_REQUIRE(ctx, kv->elem == MB_KV_BF16 || kv->elem == MB_KV_NVFP4, "%s: pages hold bf16 or NVFP4 rows, not element type %d",
             what, kv->elem);
  MB_REQUIRE(ctx, kv->d == 64 || kv->d == 128, "%s: head_dim must be 64 or 128, got %zu", what, kv->d);
  MB_REQUIRE(ctx, kv->page_size >= 16 && kv->page_size % 16 == 0 && kv->page_size <= (1u << 20),
             "%s: the page size must be a multiple of 16 (up to 2^20), got %zu", what, kv->page_size);
  MB_REQUIRE(ctx, kv->batch > 0 && kv->batch <= 65535 && kv->kv_heads > 0 && kv->kv_heads <= 4096 && kv->pages > 0 &&
                      kv->pages < (1ull << 31),
             "%s: bad extents (batch %zu, kv_heads %zu, pages %zu)", what, kv->batch, kv->kv_heads, kv->pages);
  MB_REQUIRE(ctx, kv->table_width > 0 && kv->table_width <= kv->table_stride && kv->table_width * kv->page_size < (1ull << 30) &&
                      kv->table_width < (1ull << 30),
             "%s: a table row of %zu pages of %zu rows (stride %zu)", what, kv->table_width, kv->page_size, kv->table_stride);
  MB_REQUIRE(ctx, heads > 0 && heads <= 65535 && heads % kv->kv_heads == 0, "%s: %zu query heads over %zu KV heads", what, heads,
             kv->kv_heads);
  MB_REQUIRE(ctx, mb_aligned(kv->k, 16) && mb_aligned(kv->v, 16) && mb_aligned(kv->block_table, 4) && mb_aligned(kv->lens, 4),
             "%s: pools need 16-byte alignment", what);
  if (kv->elem == MB_KV_NVFP4)
    MB_REQUIRE(ctx, kv->k_scales && kv->v_scales && mb_aligned(kv->k_scales, 8) && mb_aligned(kv->v_scales, 8),
               "%s: NVFP4 pools need 8-byte aligned scales", what);
  if (terms) {
    MB_REQUIRE(ctx, terms->scale > 0.0f && terms->scale <= 1.0e18f, "%s: scale must be positive and at most 1e18", what);
    MB_REQUIRE(ctx, terms->softcap >= 0.0f && terms->softcap <= 1.0e18f, "%s: softcap must be zero (none) or positive and at most 1e18",
               what);
    MB_REQUIRE(ctx, terms->softcap == 0.0f || terms->scale / terms->softcap <= 3.0e38f, "%s: softcap %g is too small for the scale", what,
               double(terms->softcap));
    MB_REQUIRE(ctx, mb_aligned(terms->slopes, 4) && mb_aligned(terms->prefix, 4), "%s: slopes and prefix need 4-byte alignment", what);
  }
  MB_REQUIRE_DEVICE(ctx, what);
  out->table = kv->block_table;
  out->lens = kv->lens;
  out->prefix = terms ? terms->prefix : nullptr;
  out->batch = uint32_t(kv->batch);
  out->pages = uint32_t(kv->pages);
  out->page_size = uint32_t(kv->page_size);
  out->kv_heads = uint32_t(kv->kv_heads);
  out->table_width = uint32_t(kv->table_width);
  out->table_stride = kv->table_stride;
  out->page_div = mb_fastdiv_make(uint32_t(kv->page_size));
  out->rows_max = uint32_t(kv->table_width * kv->page_size);
  // no row is further away than the table reaches, so a wider window is none
  out->window = terms && terms->window < out->rows_max ? uint32_t(terms->window) : 0;
  out->plan_flag = ctx->flags_dev ? ctx->flags_dev + MB_FLAG_PLAN_FAULT : nullptr;
  return MB_OK;
}

MB_API int mb_paged_append(mb_ctx* ctx, mb_stream stream_, const void* qkv, size_t qkv_stride, size_t tokens, size_t hq,
                           const mb_paged_kv* kv, const int32_t* cu_q, const float* inv_freq, const int32_t* positions,
                           size_t axes, const int32_t* section_end, void* q_out) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  AppendParams p;
  int rc = paged_view(ctx, "paged_append", kv, nullptr, kv ? kv->kv_heads : 1, &p.c);
  if (rc) return rc;
  MB_REQUIRE(ctx, inv_freq && (tokens == 0 || (qkv && q_out)), "paged_append: null argument");
  MB_REQUIRE(ctx, hq > 0 && hq <= 65535, "paged_append: bad query head count %zu", hq);
  const size_t heads = hq + 2 * kv->kv_heads;
  MB_REQUIRE(ctx, qkv_stride >= heads * kv->d && qkv_stride % 8 == 0,
             "paged_append: rows of %zu values %zu apart (a multiple of 8 is needed)", heads * kv->d, qkv_stride);
  MB_REQUIRE(ctx, tokens < (1ull << 31), "paged_append: too many tokens");
  MB_REQUIRE(ctx, cu_q || tokens % kv->batch == 0, "paged_append: %zu tokens do not divide among %zu sequences", tokens, kv->batch);
  MB_REQUIRE(ctx, mb_aligned(qkv, 16) && mb_aligned(q_out, 16) && mb_aligned(inv_freq, 4) && mb_aligned(positions, 4) &&
                      mb_aligned(cu_q, 4),
             "paged_append: 16-byte alignment");
  if (positions) {
    MB_REQUIRE(ctx, axes >= 1 && axes <= 4 && section_end, "paged_append: one to four position axes with their sections, got %zu", axes);
    for (size_t a = 0; a < axes; ++a)
      MB_REQUIRE(ctx, section_end[a] >= (a ? section_end[a - 1] : 0) && section_end[a] <= int32_t(kv->d / 2),
                 "paged_append: section ends must ascend to d / 2");
    MB_REQUIRE(ctx, section_end[axes - 1] == int32_t(kv->d / 2), "paged_append: the sections must cover d / 2 = %zu frequencies",
               kv->d / 2);
  }
  if (tokens == 0) return MB_OK;
  p.qkv = static_cast<const uint4*>(qkv);
  p.q_out = static_cast<uint4*>(q_out);
  p.k = kv->k; p.v = kv->v; p.ks = kv->k_scales; p.vs = kv->v_scales;
  p.cu_q = cu_q; p.positions = positions; p.inv_freq = inv_freq;
  p.tokens = uint32_t(tokens); p.per_seq = uint32_t(cu_q ? 1 : tokens / kv->batch);
  p.hq = uint32_t(hq); p.heads = uint32_t(heads);
  p.stride16 = qkv_stride / 8;
  p.axes = uint32_t(positions ? axes : 1);
  for (size_t a = 0; a < 4; ++a) p.section_end[a] = positions && a < axes ? uint32_t(section_end[a]) : uint32_t(kv->d / 2);
  // Tokens of a block: one keeps a short call's chain short and its grid wide, four share the block's set-up (bf16 pages, 32
  // query and 8 KV heads of 128, one / four: 3.3 / 4.7 us at 64 tokens, 6.9 / 7.1 at 1024, 10.1 / 11.0 at 2048, 19.8 / 19.4
  // at 4096).
  const bool fp4 = kv->elem == MB_KV_NVFP4, wide = tokens >= 4096;
  dim3 grid(unsigned(wide ? (tokens + 3) / 4 : tokens), 1);
  cudaError_t e = fp4 ? (wide ? launch_append<true, 4>(p, uint32_t(kv->d), grid, stream) : launch_append<true, 1>(p, uint32_t(kv->d), grid, stream))
                      : (wide ? launch_append<false, 4>(p, uint32_t(kv->d), grid, stream) : launch_append<false, 1>(p, uint32_t(kv->d), grid, stream));
  MB_CUDA_OK(ctx, e);
  MB_LAUNCH_OK(ctx);
  return MB_OK;
}

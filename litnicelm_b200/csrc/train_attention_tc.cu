// Attention with its backward pass for training on the sm_100a tensor cores (tcgen05 + TMEM + TMA): bfloat16 operands, 32-bit
// scores, weights' sums, statistics and accumulators. The mathematics is that of train_attention.cu.
//
// forward   one CTA per 128 rows of a head walks the tiles of 128 keys they see: S = Q K^T, four warps (a thread: a row) turn S
//           into weights 2^(s - m), stored as bfloat16 over the scores' own columns of tensor memory, O += P V from there. The
//           reference m follows a row's maximum only where that has grown by more than 2^8, so most tiles need no pass over O.
//           Two CTAs share an SM: one's products run under the other's softmax. Up to 64 dimensions one CTA with two tiles of rows
//           and its scores, weights and sums apart in tensor memory instead.
// dk, dv    one CTA per 128 keys of a key head walks the tiles of 128 rows that see them, through all query heads that share it:
//           S^T = K Q^T, dP^T = V dO^T; eight warps (a thread: a key and half of the rows) make P^T and then dS^T = P^T (dP^T -
//           delta), each over its source's columns; dV += P^T dO and dK += dS^T Q with A from tensor memory and B as it lies in
//           shared memory, rows of k. While the warps work on P the pipe multiplies for dS of the tile before, and the
//           other way round: dV(i), S(i+1) | dK(i), dP(i+1); at 64 dimensions a third tile fits into tensor memory, and each product
//           for the warps is issued one step sooner.
// dq        one CTA per 128 rows of a head in the same way: S = Q K^T, dP = dO V^T, dQ += dS K, with two places for dP.
// These kernels (but the forward of 128 dimensions, whose two CTAs do that for each other) stay on their SM: a CTA takes over blocks that
// have not started (TtNext), so that the next tile's operands and first products arrive under the last one's results.
//
// Bound, 4 streams of 2048 rows, 16 heads of 64, causal (forward 65, delta 12, dq 81, dk and dv 103 us): the exponentials, 16 a clock and
// SM, are 32 us of each kernel, the products 24 us of the forward, 32 of dq, 48 of dk and dv (those into 64 columns take as long as into
// 128); a tile's stages - product, softmax, product - wait for one another, and what two tiles in flight do not hide is the
// rest. 8192 rows of 16 heads of 128 on 4 key heads (forward 253, delta 21, dq 323, dk and dv 455 us in the
// first passes, together 1.05 ms; from about the hundredth in a row on 287, 23, 363 and 494): 121 us of exponentials, products of 121, 182
// and 242 us; the largest of the 256 blocks for dk and dv holds 256 of the 225 tiles that an SM has on average.
// The scores are computed once for each, so that no sum depends on the order in which CTAs finish.
//
// Rounding to bfloat16: P and dS for their products (the tensor cores take both operands of one type), relative 2^-8 a term,
// of independent sign, as much as the operands themselves have been rounded by; the results.
//
// Warp 0 issues TMA, warp 1 owns tensor memory and issues the MMAs. Rows outside the tensors load as zeros; keys behind a
// stream's length or every row, and rows that see no key, are cleared in shared memory where a product would multiply them by a weight of
// zero. Every wait is bounded; one that runs out ends the CTA, whose results are then NaN. No clusters, no multicast.
#include "train_attention_tc.cuh"

namespace lb {

namespace {

constexpr int TT_FWD_THREADS = 192, TT_BWD_THREADS = 320;

// One row's columns c0 .. c0 + 15 of a result, as bfloat16.
__device__ __forceinline__ void tt_store16(bf16 *row, const TtArgs &a, int c0, const float (&x)[16]) {
  if (a.vec && c0 + 16 <= a.dim) {
    unsigned w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = tt_pack(x[2 * j], x[2 * j + 1]);
    *reinterpret_cast<uint4 *>(row + c0) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4 *>(row + c0 + 8) = make_uint4(w[4], w[5], w[6], w[7]);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (c0 + j < a.dim) row[c0 + j] = __float2bfloat16_rn(x[j]);
  }
}

// Accumulator columns [c0, c1) of this thread's lane times `factor` into its row of a result; NaN where the CTA gave up.
__device__ __forceinline__ void tt_store_row(bf16 *row, bool live, const TtArgs &a, unsigned tmem, int c0, int c1, float factor,
                                             bool zero, bool ok) {
#pragma unroll 1
  for (int c = c0; c < c1; c += 16) {
    float x[16];
    if (ok && !zero) {
      unsigned r[16];
      tc_ld16(tmem + (unsigned)c, r);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = __uint_as_float(r[j]) * factor;
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = ok ? 0.f : NAN;
    }
    if (live) tt_store16(row, a, c, x);
  }
}

// A tile of 128 rows from r0 on of a head's result, as zeros (by one warp).
__device__ __forceinline__ void tt_store_zeros(const HeadView &o, const TtArgs &a, const TtPlace &at, int r0, int rows, int lane) {
  const float none[16] = {};
  for (int row = r0 + lane; row < min(r0 + TT_B, rows); row += 32)
    for (int c = 0; c < a.dim; c += 16)
      tt_store16(reinterpret_cast<bf16 *>(o.p) + at.stream * o.s + (long long)row * o.r + at.head * o.h, a, c, none);
}

// Rows `from` .. 127 of a tile of slabs, as zeros (by one warp; the tensor cores read them next).
__device__ __forceinline__ void tt_clear_rows(unsigned char *tile, int slabs, int from, int lane) {
  for (int s = 0; s < slabs; ++s)
    for (int e = from * 8 + lane; e < 128 * 8; e += 32)
      *reinterpret_cast<uint4 *>(tile + s * TT_SLAB + e * 16) = make_uint4(0u, 0u, 0u, 0u);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}

// 2^x of both halves. (Of a quarter of them by a polynomial on the FMA pipe, as the unit that this instruction runs on takes 1024 clocks
// a tile: forward 75 -> 80 us, dq and dkv 2 % less, at D = 128 10 % more. So not.)
__device__ __forceinline__ unsigned long long tt_exp2_two(unsigned long long x) { return tt_two(tt_exp2(tt_lo(x)), tt_exp2(tt_hi(x))); }

// S (128 x 128) = rows of a . rows of b over dim, both with contiguous dim. The loops that issue products are unrolled, with
// descriptors that differ by constants: with a loop over the steps that dim needs, each instruction's descriptors took the one
// issuing thread about 130 clocks, twice what the tensor pipe takes for the product.
template <int D>
__device__ __forceinline__ void tt_mma_rows(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc) {
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) {
    const unsigned long long at = (unsigned long long)((ks >> 2) * (TT_SLAB >> 4) + (ks & 3) * 2);
    tc_mma_f16(d, a + at, b + at, idesc, ks ? 1u : 0u);
  }
}
// d (+)= weights in tensor memory (columns from w on; HALVES: two groups of 32, 64 apart) . rows of b, 128 of k
template <bool HALVES>
__device__ __forceinline__ void tt_mma_weights(unsigned d, unsigned w, unsigned long long b, unsigned idesc, bool more) {
#pragma unroll
  for (int ks = 0; ks < TT_B / 16; ++ks)
    tc_mma_f16_ts(d, w + (unsigned)(HALVES ? (ks >> 2) * 64 + (ks & 3) * 8 : ks * 8), b + (unsigned long long)(ks * (16 * 128 >> 4)),
                  idesc, ks ? 1u : (unsigned)more);
}
// Descriptors of a tile: rows along k, and rows of k.
__device__ __forceinline__ unsigned long long tt_rows(unsigned tile) { return umma_desc_k128(tile); }
__device__ __forceinline__ unsigned long long tt_cols(unsigned tile) { return umma_desc_mn128(tile, TT_SLAB); }

// A row's scores of a tile (128 registers) to its new reference m; keep: what its sums are worth under it.
__device__ __forceinline__ bool tt_reference(float (&s)[TT_B], const TtArgs &a, float factor, bool inside, int c_lo, int c_end, float &m,
                                             float &l, float &keep) {
  if (a.factor < 0.f) {
#pragma unroll
    for (int j = 0; j < TT_B; ++j) s[j] = -s[j];
  }
  if (!inside) {
#pragma unroll
    for (int j = 0; j < TT_B; ++j)
      if (j >= c_end || j < c_lo) s[j] = -INFINITY;
  }
  float mq[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
  for (int j = 4; j < TT_B; j += 4) {
    if ((j >> 2) & 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) mq[e] = tt_max3(mq[e], s[j + e], j + 4 < TT_B ? s[(j + 4 + e) % TT_B] : s[j + e]);
    }
  }
  const float top = tt_max3(tt_max3(mq[0], mq[1], mq[2]), mq[3], mq[3]) * factor;
  const float mx = fmaxf(TT_NEG, top);
  const bool grow = mx > m + TT_SLACK;
  keep = grow ? tt_exp2(m - mx) : 1.f;
  if (grow) m = mx;
  if (top != top) m = top;  // a score that is no number, or infinite, shows in the reference, and so in the sum
  l *= keep;
  return grow;
}
// The weights 2^(factor s - m), summed into l, as bfloat16 over the scores' own columns, which this warp has read.
__device__ __forceinline__ void tt_weights(const float (&s)[TT_B], float factor, float m, float &l, unsigned tmem) {
  unsigned long long lq[4] = {0ull, 0ull, 0ull, 0ull};
  const unsigned long long f2 = tt_two(factor, factor), m2 = tt_two(-m, -m);
#pragma unroll
  for (int c0 = 0; c0 < TT_B; c0 += 32) {
    unsigned pk[16];
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      const unsigned long long e = tt_exp2_two(tt_fma2(tt_two(s[c0 + j], s[c0 + j + 1]), f2, m2));
      lq[(j >> 1) & 3] = tt_add2(lq[(j >> 1) & 3], e);
      pk[j >> 1] = tt_pack(tt_lo(e), tt_hi(e));
    }
    tc_st16(tmem + (unsigned)(c0 >> 1), pk);
  }
  lq[0] = tt_add2(tt_add2(lq[0], lq[1]), tt_add2(lq[2], lq[3]));
  l += tt_lo(lq[0]) + tt_hi(lq[0]);
}
// m is rounded, factor s - m is not until it is an exponent: a factor of 2^(|m| 2^-25) common to a row's weights, which cancels, but far
// from zero is more than 32 bits hold. Such a row is computed again when its tiles are done, by one warp, a lane a key, in 32-bit
// arithmetic with rounded scores. (With the scores of a tile rounded first where a reference is far, the branch alone took the forward
// of 4 x 2048 rows from 63.6 to 67.5 us.)
__device__ __forceinline__ bool tt_far(float m, float l) {
  return fabsf(m) < INFINITY && (fabsf(m) > TT_FAR || !(l > 0.f && l < INFINITY));
}
__device__ __noinline__ void tt_row_again(const TtArgs &a, int stream, int head, int row, int lo, int end, int lane) {
  const int kh = head / a.share;
  const bf16 *q = reinterpret_cast<const bf16 *>(a.q.p) + stream * a.q.s + (long long)row * a.q.r + head * a.q.h;
  const bf16 *k = reinterpret_cast<const bf16 *>(a.k.p) + stream * a.k.s + kh * a.k.h;
  const bf16 *v = reinterpret_cast<const bf16 *>(a.v.p) + stream * a.v.s + kh * a.v.h;
  auto score = [&](int j) {
    const bf16 *x = k + (long long)j * a.k.r;
    float s = 0.f;
    for (int c = 0; c < a.dim; c += 8) {  // (what TMA can address: dim a multiple of 8, rows on 16-byte boundaries)
      const uint4 u = *reinterpret_cast<const uint4 *>(q + c), w = *reinterpret_cast<const uint4 *>(x + c);
      const __nv_bfloat162 *y = reinterpret_cast<const __nv_bfloat162 *>(&u), *z = reinterpret_cast<const __nv_bfloat162 *>(&w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __bfloat1622float2(y[i]), g = __bfloat1622float2(z[i]);
        s = fmaf(f.x, g.x, fmaf(f.y, g.y, s));
      }
    }
    return __fmul_rn(s, a.factor);  // (rounded, or the difference from m is not)
  };
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j = lo + lane; j < end; j += 32) m = fmaxf(m, score(j));
  for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
  for (int j0 = lo; j0 < end; j0 += 32) {
    const float p = j0 + lane < end ? tt_exp2(score(j0 + lane) - m) : 0.f;
    l += p;
#pragma unroll 4
    for (int t = 0; t < min(32, end - j0); ++t) {
      const float w = __shfl_sync(0xffffffffu, p, t);
      const bf16 *x = v + (long long)(j0 + t) * a.v.r;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (lane + 32 * e < a.dim) o[e] = fmaf(w, __bfloat162float(x[lane + 32 * e]), o[e]);
    }
  }
  for (int i = 16; i > 0; i >>= 1) l += __shfl_xor_sync(0xffffffffu, l, i);
  bf16 *out = reinterpret_cast<bf16 *>(a.o1.p) + stream * a.o1.s + (long long)row * a.o1.r + head * a.o1.h;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (lane + 32 * e < a.dim) out[lane + 32 * e] = __float2bfloat16_rn(o[e] / l);
  if (lane == 0) a.lse[((long long)stream * a.heads + head) * a.n + row] = (m + log2f(l)) * 0.6931471805599453f;
}
// Those of a warp's 32 rows from row0 on, behind what the tiles have left of them.
__device__ __forceinline__ void tt_rows_again(const TtArgs &a, const TtPlace &at, int row0, unsigned which, int lane) {
  __syncwarp();
  for (; which != 0u; which &= which - 1u) {
    const int row = row0 + __ffs((int)which) - 1;
    tt_row_again(a, at.stream, at.head, row, a.span.lo(row), a.span.end(row, at.keys), lane);
  }
}

// This lane's accumulator row times keep.
__device__ __forceinline__ void tt_rescale(unsigned tmem, int dim, float keep) {
#pragma unroll 1
  for (int c0 = 0; c0 < dim; c0 += 16) {
    unsigned r[16];
    tc_ld16(tmem + (unsigned)c0, r);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * keep);
    tc_st16(tmem + (unsigned)c0, r);
  }
}

template <int D>
__global__ void __launch_bounds__(TT_FWD_THREADS, 2)
train_forward_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TtArgs a) {
  constexpr int SLABS = D / 64, TILE = SLABS * TT_SLAB;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const unsigned base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char *base_ptr = smem_raw + (base - smem_u32(smem_raw));
  const unsigned q_off = base, k_off = base + TILE, v_off = base + 2 * TILE, bars = base + 3 * TILE;
  const unsigned q_full = bars, k_full = bars + 8, v_full = bars + 16, k_free = bars + 24, s_full = bars + 32,
                 p_ready = bars + 40, o_full = bars + 48, drained = bars + 56;
  volatile unsigned *tmem_holder = reinterpret_cast<volatile unsigned *>(base_ptr + 3 * TILE + 64);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(base_ptr + 3 * TILE + 68);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const TtPlace at = tt_place(a, a.heads, a.span.causal != 0);
  const int r0 = at.tile * TT_B, r1 = min(r0 + TT_B, a.n), kh = at.head / a.share;
  const int lo = a.span.lo(r0), end = a.span.end(r1 - 1, at.keys);
  const int tiles = end > lo ? (end - lo + TT_B - 1) / TT_B : 0;

  if (threadIdx.x == 0) {
    for (unsigned bar : {q_full, k_full, v_full, k_free, s_full, o_full, drained}) mbar_init(bar, 1);
    mbar_init(p_ready, 4);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) tt_alloc(tmem_holder, 256u);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned tmem_s = *tmem_holder, tmem_o = tmem_s + TT_B;

  if (warp == 0) {
    int k_loads = 0, v_loads = 0;
    bool ok = true;
    if (lane == 0 && tiles > 0) {
      mbar_expect_tx(q_full, (unsigned)TILE);
      for (int s = 0; s < SLABS; ++s) tma_load_4d(q_off + s * TT_SLAB, &map_q, s * 64, at.head, r0, at.stream, q_full);
    }
    for (int i = 0; i < tiles && ok; ++i) {
      const int j0 = lo + i * TT_B;
      if (i > 0) ok = mbar_wait(k_free, (unsigned)(i - 1) & 1u, abort_flag, nullptr, 71);
      __syncwarp();
      if (!ok) break;
      if (lane == 0) {
        mbar_expect_tx(k_full, (unsigned)TILE);
        for (int s = 0; s < SLABS; ++s) tma_load_4d(k_off + s * TT_SLAB, &map_k, s * 64, kh, j0, at.stream, k_full);
      }
      ++k_loads;
      if (i > 0) ok = mbar_wait(o_full, (unsigned)(i - 1) & 1u, abort_flag, nullptr, 72);  // P V has read the values
      __syncwarp();
      if (!ok) break;
      if (lane == 0) {
        mbar_expect_tx(v_full, (unsigned)TILE);
        for (int s = 0; s < SLABS; ++s) tma_load_4d(v_off + s * TT_SLAB, &map_v, s * 64, kh, j0, at.stream, v_full);
      }
      ++v_loads;
      __syncwarp();
    }
    if (*abort_flag && tiles > 0) {  // copies in flight must land before the shared memory goes away
      const unsigned long long limit = global_timer() + WAIT_LIMIT_NS;
      while (!mbar_try_wait(q_full, 0) && global_timer() < limit) {}
      while (k_loads > 0 && !mbar_try_wait(k_full, (unsigned)(k_loads - 1) & 1u) && global_timer() < limit) {}
      while (v_loads > 0 && !mbar_try_wait(v_full, (unsigned)(v_loads - 1) & 1u) && global_timer() < limit) {}
    }
  } else if (warp == 1) {
    const int cols = (a.dim + 15) & ~15;
    const unsigned long long q_rows = tt_rows(q_off), k_rows = tt_rows(k_off), v_cols = tt_cols(v_off);
    const unsigned idesc_s = umma_idesc_bf16(TT_B), idesc_o = umma_idesc_bf16(cols) | UMMA_B_MN_MAJOR;
    bool ok = tiles > 0 ? mbar_wait_warp(q_full, 0, abort_flag, nullptr, 73) : true;
    int i = 0;
    for (; i < tiles && ok; ++i) {
      ok = mbar_wait_warp(k_full, (unsigned)i & 1u, abort_flag, nullptr, 74);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (tc_elect()) {
        tt_mma_rows<D>(tmem_s, q_rows, k_rows, idesc_s);
        tc_commit(k_free);
        tc_commit(s_full);
      }
      __syncwarp();
      ok = mbar_wait_warp(v_full, (unsigned)i & 1u, abort_flag, nullptr, 75);
      if (!ok) break;
      const int have = at.keys - (lo + i * TT_B);
      if (have < TT_B && at.keys < a.m) tt_clear_rows(base_ptr + 2 * TILE, SLABS, have, lane);
      ok = mbar_wait_warp(p_ready, (unsigned)i & 1u, abort_flag, nullptr, 76);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (tc_elect()) {
        tt_mma_weights<false>(tmem_o, tmem_s, v_cols, idesc_o, i > 0);
        tc_commit(o_full);
      }
      __syncwarp();
    }
    if (!ok) {  // a bounded chance for the tensor pipe to finish before tensor memory is freed (a barrier that no one else waits for)
      if (tc_elect()) tc_commit(drained);
      __syncwarp();
      const unsigned long long limit = global_timer() + WAIT_LIMIT_NS;
      while (!mbar_try_wait(drained, 0) && global_timer() < limit) {}
    }
  } else {
    const int q = warp & 3;
    const unsigned lanes = (unsigned)(q * 32) << 16;
    const int row = r0 + q * 32 + lane;
    const int row_lo = a.span.lo(row), row_end = a.span.end(row, at.keys);
    const int warp_lo = a.span.lo(r0 + q * 32 + 31), warp_end = a.span.end(r0 + q * 32, at.keys);
    // a negative factor's sign goes to the scores; zero is small, so that hidden scores of -infinity stay that
    const float factor = fmaxf(fabsf(a.factor), 1e-30f);
    float m = TT_NEG, l = 0.f;
    bool ok = true;
    for (int i = 0; i < tiles && ok; ++i) {
      const int j0 = lo + i * TT_B;
      ok = mbar_wait_warp(s_full, (unsigned)i & 1u, abort_flag, nullptr, 77);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int c_lo = row_lo - j0, c_end = row_end - j0;  // keys j0 + c that this row sees
      const bool inside = warp_lo <= j0 && warp_end >= j0 + TT_B;
      float s[TT_B];
      {
        unsigned(&u)[4][32] = reinterpret_cast<unsigned(&)[4][32]>(s);
#pragma unroll
        for (int c = 0; c < 4; ++c) tc_ld32(tmem_s + lanes + (unsigned)(c * 32), u[c]);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      }
      float keep;
      const bool grow = tt_reference(s, a, factor, inside, c_lo, c_end, m, l, keep);
      // (the scores are there, so the product before them is done)
      if (i > 0 && __any_sync(0xffffffffu, grow)) tt_rescale(tmem_o + lanes, a.dim, keep);
      tt_weights(s, factor, m, l, tmem_s + lanes);
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready);
    }
    if (ok && tiles > 0) ok = mbar_wait_warp(o_full, (unsigned)(tiles - 1) & 1u, abort_flag, nullptr, 79);
    ok = __all_sync(0xffffffffu, ok && !*abort_flag);
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const bool live = row < a.n, empty = row_end <= row_lo;
    bf16 *o = reinterpret_cast<bf16 *>(a.o1.p) + at.stream * a.o1.s + (long long)row * a.o1.r + at.head * a.o1.h;
    // a warp's rows are read together: a row without keys has factor 0 (its accumulator holds finite weights of nothing)
    const float inv = empty ? 0.f : 1.0f / l;
    tt_store_row(o, live, a, tmem_o + lanes, 0, (a.dim + 15) & ~15, inv, tiles == 0, ok);
    if (live)
      a.lse[((long long)at.stream * a.heads + at.head) * a.n + row] =
          !ok ? NAN : empty ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
    const unsigned far = __ballot_sync(0xffffffffu, ok && live && !empty && tt_far(m, l));
    if (far != 0u) tt_rows_again(a, at, r0 + q * 32, far, lane);
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_s), "r"(256u));
  }
}

// The same for heads of up to 64 dimensions and more than 128 rows: one CTA per SM takes two tiles of 128 rows, A and B, with four warps
// each, and walks the tiles of keys once for both. Tensor memory holds a tile of scores, its weights and an accumulator for each, so that
// a group's next scores are made as soon as its warps have the last ones in registers, and are there before it has finished with
// those. (With two CTAs of one tile, weights over the scores, a group waited 1000 of its 3400 clocks a tile for them; with three
// places that jobs A0 B0 A1 B1 .. took in turn, each waited for the other's product.) Blocks go on with the next rows (TtNext).
constexpr int TT_PAIR_STAGES = 4;
constexpr int TT_PAIR_BAR = (4 + 2 * TT_PAIR_STAGES) * TT_SLAB, TT_PAIR_SMEM = TT_PAIR_BAR + 384 + 1024;

__global__ void __launch_bounds__(TT_BWD_THREADS, 1)
train_forward_pair_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                          const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TtArgs a) {
  constexpr int NS = TT_PAIR_STAGES;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const unsigned base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char *base_ptr = smem_raw + (base - smem_u32(smem_raw));
  const unsigned bars = base + TT_PAIR_BAR;
  auto q_tile = [&](int s) { return base + (unsigned)(s * 2 * TT_SLAB); };  // of A, and of B behind it
  auto k_tile = [&](int s) { return base + (unsigned)((4 + s) * TT_SLAB); };
  auto v_tile = [&](int s) { return base + (unsigned)((4 + NS + s) * TT_SLAB); };
  auto k_full = [&](int s) { return bars + 8u * s; };
  auto k_empty = [&](int s) { return bars + 32u + 8u * s; };
  auto v_full = [&](int s) { return bars + 64u + 8u * s; };
  auto v_empty = [&](int s) { return bars + 96u + 8u * s; };
  auto s_full = [&](int group) { return bars + 128u + 8u * group; };
  auto s_read = [&](int group) { return bars + 144u + 8u * group; };
  auto p_ready = [&](int group) { return bars + 160u + 8u * group; };
  auto o_full = [&](int group) { return bars + 176u + 8u * group; };
  auto q_full = [&](int s) { return bars + 192u + 8u * s; };
  auto q_empty = [&](int s) { return bars + 208u + 8u * s; };
  volatile unsigned *tmem_holder = reinterpret_cast<volatile unsigned *>(base_ptr + TT_PAIR_BAR + 224);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(base_ptr + TT_PAIR_BAR + 228);
  TtNext next{bars + 256u};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s)
      for (unsigned bar : {k_full(s), k_empty(s), v_full(s), v_empty(s)}) mbar_init(bar, 1);
    for (int s = 0; s < 2; ++s) {
      for (unsigned bar : {s_full(s), o_full(s), q_full(s), q_empty(s)}) mbar_init(bar, 1);
      mbar_init(s_read(s), 4);
      mbar_init(p_ready(s), 4);
    }
    next.init(9);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) tt_alloc(tmem_holder, 512u);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned tmem = *tmem_holder;

  struct Item {
    TtPlace at;
    int r0, lo, tiles_a, tiles_b;
    __device__ int tiles() const { return max(tiles_a, tiles_b); }
  };
  auto item = [&](int block) {
    Item x;
    x.at = tt_place(a, a.heads, a.span.causal != 0, 1, block);
    x.r0 = x.at.tile * 2 * TT_B;
    x.lo = a.span.lo(x.r0);
    auto tiles_of = [&](int first) {
      const int end = first < a.n ? a.span.end(min(first + TT_B, a.n) - 1, x.at.keys) : 0;
      return end > x.lo ? (end - x.lo + TT_B - 1) / TT_B : 0;
    };
    x.tiles_a = tiles_of(x.r0);
    x.tiles_b = tiles_of(x.r0 + TT_B);
    return x;
  };

  if (warp == 0) {
    int it = 0, n = 0, k_loads = 0, v_loads = 0;  // tiles of keys so far, items, loads issued
    bool ok = true;
    int block = (int)blockIdx.x;
    for (int w = 0;; ++w) {
      Item x = item(max(block, 0));
      while (block >= 0 && x.tiles() == 0) {
        for (int half = 0; half < 2; ++half) tt_store_zeros(a.o1, a, x.at, x.r0 + half * TT_B, a.n, lane);
        for (int row = x.r0 + lane; row < min(x.r0 + 2 * TT_B, a.n); row += 32)
          a.lse[((long long)x.at.stream * a.heads + x.at.head) * a.n + row] = -INFINITY;
        next.ask(lane);
        block = next.answer();
        x = item(max(block, 0));
      }
      next.push(w, block, lane);
      if (block < 0) break;
      bool asked = false;
      const int kh = x.at.head / a.share, sq = n & 1, tiles = x.tiles();
      if (ok) {
        ok = mbar_wait_warp(q_empty(sq), ((unsigned)(n >> 1) & 1u) ^ 1u, abort_flag, nullptr, 60);
        if (ok && lane == 0) {
          mbar_expect_tx(q_full(sq), 2u * TT_SLAB);
          tma_load_4d(q_tile(sq), &map_q, 0, x.at.head, x.r0, x.at.stream, q_full(sq));
          tma_load_4d(q_tile(sq) + TT_SLAB, &map_q, 0, x.at.head, x.r0 + TT_B, x.at.stream, q_full(sq));
        }
        if (ok) ++n;
        __syncwarp();
      }
      for (int i = 0; i < tiles && ok; ++i, ++it) {
        const int st = it % NS, j0 = x.lo + i * TT_B;
        const unsigned free = ((unsigned)(it / NS) & 1u) ^ 1u;
        ok = mbar_wait_warp(k_empty(st), free, abort_flag, nullptr, 61);
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(k_full(st), TT_SLAB);
          tma_load_4d(k_tile(st), &map_k, 0, kh, j0, x.at.stream, k_full(st));
        }
        ++k_loads;
        __syncwarp();
        if (i + 1 == tiles) {
          next.ask(lane);
          asked = true;
        }
        ok = mbar_wait_warp(v_empty(st), free, abort_flag, nullptr, 62);
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(v_full(st), TT_SLAB);
          tma_load_4d(v_tile(st), &map_v, 0, kh, j0, x.at.stream, v_full(st));
        }
        ++v_loads;
        __syncwarp();
      }
      if (!asked) next.ask(lane);
      block = next.answer();
    }
    if (*abort_flag) {  // copies in flight must land before the shared memory goes away
      const unsigned long long limit = global_timer() + WAIT_LIMIT_NS;
      for (int j = n > 2 ? n - 2 : 0; j < n; ++j)
        while (!mbar_try_wait(q_full(j & 1), (unsigned)(j >> 1) & 1u) && global_timer() < limit) {}
      for (int j = k_loads > NS ? k_loads - NS : 0; j < k_loads; ++j)
        while (!mbar_try_wait(k_full(j % NS), (unsigned)(j / NS) & 1u) && global_timer() < limit) {}
      for (int j = v_loads > NS ? v_loads - NS : 0; j < v_loads; ++j)
        while (!mbar_try_wait(v_full(j % NS), (unsigned)(j / NS) & 1u) && global_timer() < limit) {}
    }
  } else if (warp == 1) {
    const int cols = (a.dim + 15) & ~15;
    const unsigned long long q_rows = tt_rows(q_tile(0)), k_rows = tt_rows(k_tile(0)), v_cols = tt_cols(v_tile(0));
    const unsigned idesc_s = umma_idesc_bf16(TT_B), idesc_o = umma_idesc_bf16(cols) | UMMA_B_MN_MAJOR;
    // A tile of keys of an item, for both groups. Its S are issued a tile ahead of P V, into the next item too.
    struct Round {
      int i, tiles, tiles_a, tiles_b, live, g, n;  // live: keys from the first tile's start on that exist; tile of all; item
    };
    Round lead{};
    lead.i = lead.g = lead.n = -1;
    int w = 0, sent[2] = {}, added[2] = {};
    auto advance = [&]() {
      ++lead.g;
      if (++lead.i < lead.tiles) return true;
      const int block = next.take(w++, lane);
      if (block < 0) return false;
      const Item x = item(block);
      lead.tiles_a = tt_uniform(x.tiles_a);
      lead.tiles_b = tt_uniform(x.tiles_b);
      lead.tiles = max(lead.tiles_a, lead.tiles_b);
      lead.live = tt_uniform(x.at.keys < a.m ? x.at.keys - x.lo : 0x7fffffff);
      lead.i = 0;
      ++lead.n;
      return true;
    };
    auto scores = [&](const Round &t) {
      const int st = t.g % NS, sq = t.n & 1;
      if (t.i == 0 && !mbar_wait_warp(q_full(sq), (unsigned)(t.n >> 1) & 1u, abort_flag, nullptr, 64)) return false;
      if (!mbar_wait_warp(k_full(st), (unsigned)(t.g / NS) & 1u, abort_flag, nullptr, 63)) return false;
#pragma unroll
      for (int group = 0; group < 2; ++group) {
        const bool last = group == 1 || t.i >= t.tiles_b;
        if (t.i >= (group ? t.tiles_b : t.tiles_a)) continue;
        if (sent[group] > 0 && !mbar_wait_warp(s_read(group), (unsigned)(sent[group] - 1) & 1u, abort_flag, nullptr, 70)) return false;
        ++sent[group];
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (tc_elect()) {
          tt_mma_rows<64>(tmem + (unsigned)(group * TT_B), q_rows + (unsigned long long)((sq * 2 + group) * (TT_SLAB >> 4)),
                          k_rows + (unsigned long long)(st * (TT_SLAB >> 4)), idesc_s);
          tc_commit(s_full(group));
          if (last) tc_commit(k_empty(st));
          if (last && t.i + 1 == t.tiles) tc_commit(q_empty(sq));
        }
        __syncwarp();
      }
      return true;
    };
    auto values = [&](const Round &t) {
      const int st = t.g % NS, have = t.live - t.i * TT_B;
      if (!mbar_wait_warp(v_full(st), (unsigned)(t.g / NS) & 1u, abort_flag, nullptr, 65)) return false;
      if (have < TT_B) tt_clear_rows(base_ptr + (v_tile(st) - base), 1, max(have, 0), lane);
#pragma unroll
      for (int group = 0; group < 2; ++group) {
        const bool last = group == 1 || t.i >= t.tiles_b;
        if (t.i >= (group ? t.tiles_b : t.tiles_a)) continue;
        if (!mbar_wait_warp(p_ready(group), (unsigned)added[group]++ & 1u, abort_flag, nullptr, 66)) return false;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (tc_elect()) {
          tt_mma_weights<false>(tmem + (unsigned)(384 + group * 64), tmem + (unsigned)(256 + group * 64),
                                v_cols + (unsigned long long)(st * (TT_SLAB >> 4)), idesc_o, t.i > 0);
          tc_commit(o_full(group));
          if (last) tc_commit(v_empty(st));
        }
        __syncwarp();
      }
      return true;
    };
    bool more = advance(), ok = !more || scores(lead);
    while (more && ok) {
      const Round now = lead;
      more = advance();
      ok = (!more || scores(lead)) && values(now);
    }
    if (!ok) {  // a bounded chance for the tensor pipe to finish before tensor memory is freed; the items' order goes on
      while (more) more = next.take(w++, lane) >= 0;
      if (tc_elect()) tc_commit(next.drained());
      __syncwarp();
      const unsigned long long limit = global_timer() + WAIT_LIMIT_NS;
      while (!mbar_try_wait(next.drained(), 0) && global_timer() < limit) {}
    }
  } else {
    const int q = warp & 3, group = (warp - 2) >> 2;
    const unsigned lanes = (unsigned)(q * 32) << 16, tmem_s = tmem + (unsigned)(group * TT_B) + lanes,
                   tmem_p = tmem + (unsigned)(256 + group * 64) + lanes, tmem_o = tmem + (unsigned)(384 + group * 64) + lanes;
    // a negative factor's sign goes to the scores; zero is small, so that hidden scores of -infinity stay that
    const float factor = fmaxf(fabsf(a.factor), 1e-30f);
    int tile = 0, done = 0;  // tiles of this group so far, products of them that it has waited for
    bool ok = true;
    int block = next.take(0, lane);
    for (int w = 1; block >= 0; ++w) {
      int mine, row_lo, row_end, warp_lo, warp_end;  // keys from the first tile's start on
      {
        const Item x = item(block);
        const int first = x.r0 + group * TT_B + q * 32;
        mine = group ? x.tiles_b : x.tiles_a;
        row_lo = a.span.lo(first + lane) - x.lo;
        row_end = a.span.end(first + lane, x.at.keys) - x.lo;
        warp_lo = a.span.lo(first + 31) - x.lo;
        warp_end = a.span.end(first, x.at.keys) - x.lo;
      }
      float m = TT_NEG, l = 0.f;
      for (int i = 0; i < mine && ok; ++i) {
        const int j0 = i * TT_B;
        ok = mbar_wait_warp(s_full(group), (unsigned)tile++ & 1u, abort_flag, nullptr, 67);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const int c_lo = row_lo - j0, c_end = row_end - j0;  // keys j0 + c that this row sees
        const bool inside = warp_lo <= j0 && warp_end >= j0 + TT_B;
        float s[TT_B], keep;
        {
          unsigned(&u)[4][32] = reinterpret_cast<unsigned(&)[4][32]>(s);
#pragma unroll
          for (int c = 0; c < 4; ++c) tc_ld32(tmem_s + (unsigned)(c * 32), u[c]);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(s_read(group));
        const bool grow = tt_reference(s, a, factor, inside, c_lo, c_end, m, l, keep);
        if (i > 0) {  // the product before has read the weights' place, and added to what may be rescaled
          ok = mbar_wait_warp(o_full(group), (unsigned)done++ & 1u, abort_flag, nullptr, 68);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (__any_sync(0xffffffffu, grow)) tt_rescale(tmem_o, a.dim, keep);
        }
        tt_weights(s, factor, m, l, tmem_p);
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready(group));
      }
      asm volatile("" : "+r"(block));  // the block's place once more, instead of in registers through the loop
      const Item x = item(block);
      const int row = x.r0 + group * TT_B + q * 32 + lane;
      block = next.take(w, lane);
      if (ok && mine > 0) ok = mbar_wait_warp(o_full(group), (unsigned)done++ & 1u, abort_flag, nullptr, 69);
      ok = __all_sync(0xffffffffu, ok && !*abort_flag);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const bool live = row < a.n, empty = row_end <= row_lo;
      bf16 *o = reinterpret_cast<bf16 *>(a.o1.p) + x.at.stream * a.o1.s + (long long)row * a.o1.r + x.at.head * a.o1.h;
      tt_store_row(o, live, a, tmem_o, 0, (a.dim + 15) & ~15, empty ? 0.f : 1.0f / l, mine == 0, ok);
      if (live)
        a.lse[((long long)x.at.stream * a.heads + x.at.head) * a.n + row] =
            !ok ? NAN : empty ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
      const unsigned far = __ballot_sync(0xffffffffu, ok && live && !empty && tt_far(m, l));
      if (far != 0u) tt_rows_again(a, x.at, x.r0 + group * TT_B + q * 32, far, lane);
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

// Shared memory of the backward kernels: two resident tiles, NA stages of the streamed tiles that two products a turn apart read (rows
// of q for dk, of k for dq) and NB of those that are done with sooner, statistics of the stages' rows. A load takes 1300 to 2000
// clocks: with two stages of both the products waited 700 to 1200 of a turn's 2600 (D = 64).
template <int D>
struct TtBwd {
  static constexpr int SLABS = D / 64, TILE = SLABS * TT_SLAB;
  static constexpr int NP = D == 64 ? 3 : 2;  // tiles of scores and dP in tensor memory, of the kernel for dk and dv
  static constexpr int NQ = D == 64 ? 2 : 1, NA = D == 64 ? 4 : 3, NB = D == 64 ? 4 : 2;
  static constexpr int A_OFF = 2 * NQ * TILE, B_OFF = A_OFF + NA * TILE;
  static constexpr int STAT_OFF = B_OFF + NB * TILE;  // [NB][2][128] floats
  static constexpr int BAR_OFF = STAT_OFF + NB * 2 * 128 * 4;
  static constexpr int TOTAL = BAR_OFF + 384 + 640;
  static_assert(TOTAL <= 227 * 1024, "");
};

template <int D>
__global__ void __launch_bounds__(TT_BWD_THREADS, 1)
train_dkv_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do,
                    const __grid_constant__ TtArgs a) {
  using L = TtBwd<D>;
  constexpr int SLABS = L::SLABS, TILE = L::TILE;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const unsigned base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char *base_ptr = smem_raw + (base - smem_u32(smem_raw));
  constexpr int NP = L::NP;
  const unsigned bars = base + L::BAR_OFF;
  auto k_tile = [&](int s) { return base + (unsigned)(s * 2 * TILE); };  // and the values' behind it
  auto q_tile = [&](int s) { return base + (unsigned)(L::A_OFF + s * TILE); };
  auto do_tile = [&](int s) { return base + (unsigned)(L::B_OFF + s * TILE); };
  float *stat = reinterpret_cast<float *>(base_ptr + L::STAT_OFF);
  auto a_full = [&](int s) { return bars + 8u * s; };
  auto a_empty = [&](int s) { return bars + 32u + 8u * s; };
  auto b_full = [&](int s) { return bars + 64u + 8u * s; };
  auto b_empty = [&](int s) { return bars + 96u + 8u * s; };
  auto kv_full = [&](int s) { return bars + 128u + 8u * s; };
  auto kv_empty = [&](int s) { return bars + 144u + 8u * s; };
  auto full = [&](int job) { return bars + 160u + 8u * (job % NP); };
  auto ready = [&](int job) { return bars + 184u + 8u * (job % NP); };
  auto stat_full = [&](int s) { return bars + 208u + 8u * s; };
  const unsigned done = bars + 240;
  volatile unsigned *tmem_holder = reinterpret_cast<volatile unsigned *>(base_ptr + L::BAR_OFF + 248);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(base_ptr + L::BAR_OFF + 252);
  TtNext next{bars + 256u};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(done, 1);
    for (int s = 0; s < NP; ++s) {
      mbar_init(full(s), 1);
      mbar_init(ready(s), 8);
    }
    for (int s = 0; s < L::NQ; ++s) {
      mbar_init(kv_full(s), 1);
      mbar_init(kv_empty(s), 1);
    }
    for (int s = 0; s < L::NA; ++s) {
      mbar_init(a_full(s), 1);
      mbar_init(a_empty(s), 1);
    }
    for (int s = 0; s < L::NB; ++s) {
      mbar_init(b_full(s), 1);
      mbar_init(b_empty(s), 1);
      mbar_init(stat_full(s), 1);
    }
    next.init(9);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) tt_alloc(tmem_holder, 512u);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned tmem = *tmem_holder, tmem_dv = tmem + NP * 128, tmem_dk = tmem_dv + D;
  auto place = [&](int job) { return tmem + (unsigned)(job % NP * 128); };
  pdl_wait();

  struct Item {
    TtPlace at;
    int j0, lo, each, tiles;  // rows that see a key of this tile: `each` tiles of them from lo on, for each query head
  };
  auto item = [&](int block) {
    Item x;
    x.at = tt_place(a, a.groups, false, 1, block);
    x.j0 = x.at.tile * TT_B;
    x.lo = a.span.causal ? max(0, x.j0 - a.span.first) / TT_B * TT_B : 0;
    const long long past = a.span.window > 0 ? (long long)min(x.j0 + TT_B, x.at.keys) - 1 + a.span.window - a.span.first : a.n;
    const int row_end = past < a.n ? (int)max(past, 0LL) : a.n;
    x.each = x.j0 < x.at.keys && row_end > x.lo ? (row_end - x.lo + TT_B - 1) / TT_B : 0;
    x.tiles = x.each * a.share;
    return x;
  };

  if (warp == 0) {
    int g = 0, n = 0, a_loads = 0, b_loads = 0;  // tiles of rows so far, items with any, loads issued
    bool ok = true;
    int block = (int)blockIdx.x;
    for (int w = 0;; ++w) {
      Item x = item(max(block, 0));
      while (block >= 0 && x.tiles == 0) {
        tt_store_zeros(a.o1, a, x.at, x.j0, a.m, lane);
        tt_store_zeros(a.o2, a, x.at, x.j0, a.m, lane);
        next.ask(lane);
        block = next.answer();
        x = item(max(block, 0));
      }
      next.push(w, block, lane);
      if (block < 0) break;
      bool asked = false;
      const int sk = n % L::NQ;
      if (ok) {
        ok = mbar_wait_warp(kv_empty(sk), ((unsigned)(n / L::NQ) & 1u) ^ 1u, abort_flag, nullptr, 82);
        if (ok && lane == 0) {
          mbar_expect_tx(kv_full(sk), 2u * TILE);
          for (int s = 0; s < SLABS; ++s) {
            tma_load_4d(k_tile(sk) + s * TT_SLAB, &map_k, s * 64, x.at.head, x.j0, x.at.stream, kv_full(sk));
            tma_load_4d(k_tile(sk) + TILE + s * TT_SLAB, &map_v, s * 64, x.at.head, x.j0, x.at.stream, kv_full(sk));
          }
        }
        if (ok) ++n;
        __syncwarp();
      }
      for (int i = 0, h = x.at.head * a.share, t = 0; i < x.tiles && ok; ++i, ++g) {
        const long long stats = ((long long)x.at.stream * a.heads + h) * a.n;
        const int sa = g % L::NA, st = g % L::NB, r0 = x.lo + t * TT_B;
        ok = mbar_wait_warp(a_empty(sa), ((unsigned)(g / L::NA) & 1u) ^ 1u, abort_flag, nullptr, 80);
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(a_full(sa), (unsigned)TILE);
          for (int s = 0; s < SLABS; ++s) tma_load_4d(q_tile(sa) + s * TT_SLAB, &map_q, s * 64, h, r0, x.at.stream, a_full(sa));
        }
        ++a_loads;
        __syncwarp();
        if (i + 1 == x.tiles) {
          next.ask(lane);
          asked = true;
        }
        ok = mbar_wait_warp(b_empty(st), ((unsigned)(g / L::NB) & 1u) ^ 1u, abort_flag, nullptr, 81);
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(b_full(st), (unsigned)TILE);
          for (int s = 0; s < SLABS; ++s) tma_load_4d(do_tile(st) + s * TT_SLAB, &map_do, s * 64, h, r0, x.at.stream, b_full(st));
        }
        ++b_loads;
        // a row that does not exist or sees no key has no weights: 2^(s - infinity)
#pragma unroll
        for (int e = lane; e < TT_B; e += 32) {
          const int row = r0 + e;
          const float z = row < a.n ? a.lse[stats + row] : -INFINITY;
          stat[st * 256 + e] = z == -INFINITY ? -INFINITY : -(z * TT_LOG2E);  // both with the sign that they are added with
          stat[st * 256 + 128 + e] = row < a.n ? -a.delta[stats + row] : 0.f;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(stat_full(st));
        __syncwarp();
        if (++t == x.each) {
          t = 0;
          ++h;
        }
      }
      if (!asked) next.ask(lane);
      block = next.answer();
    }
    if (*abort_flag) {  // copies in flight must land before the shared memory goes away
      const unsigned long long limit = global_timer() + WAIT_LIMIT_NS;
      for (int j = n > L::NQ ? n - L::NQ : 0; j < n; ++j)
        while (!mbar_try_wait(kv_full(j % L::NQ), (unsigned)(j / L::NQ) & 1u) && global_timer() < limit) {}
      for (int j = a_loads > L::NA ? a_loads - L::NA : 0; j < a_loads; ++j)
        while (!mbar_try_wait(a_full(j % L::NA), (unsigned)(j / L::NA) & 1u) && global_timer() < limit) {}
      for (int j = b_loads > L::NB ? b_loads - L::NB : 0; j < b_loads; ++j)
        while (!mbar_try_wait(b_full(j % L::NB), (unsigned)(j / L::NB) & 1u) && global_timer() < limit) {}
    }
  } else if (warp == 1) {
    const int cols = (a.dim + 15) & ~15;
    const unsigned long long k_rows = tt_rows(k_tile(0)), q_rows = tt_rows(q_tile(0)), do_rows = tt_rows(do_tile(0)),
                             q_cols = tt_cols(q_tile(0)), do_cols = tt_cols(do_tile(0));
    auto stage = [](int s) { return (unsigned long long)(s * (TILE >> 4)); };
    const unsigned idesc_s = umma_idesc_bf16(TT_B), idesc_d = umma_idesc_bf16(cols) | UMMA_B_MN_MAJOR;
    // Jobs: S and dP of each tile in turn, of all items; each takes the next place, and is issued behind the product that read it.
    int w = 0, i = -1, n = -1, issued = 0, tiles = 0;  // issued: tiles whose S is
    bool more = true, ok = true;
    unsigned ends = 0u;  // bit (tile of all) % 4: it is its item's last, % 4 + 4: first
    auto kv_rows = [&]() { return k_rows + (unsigned long long)(n % L::NQ * (2 * TILE >> 4)); };
    auto scores = [&]() {
      if (++i >= tiles) {
        const int block = next.take(w++, lane);
        if (block < 0) {
          more = false;
          return;
        }
        tiles = tt_uniform(item(block).tiles);
        i = 0;
        ++n;
      }
      const int g = issued, sa = g % L::NA, sk = n % L::NQ;
      const unsigned bit = 1u << (g & 3);
      ends = (ends & ~(bit | bit << 4)) | (i + 1 == tiles ? bit : 0u) | (i == 0 ? bit << 4 : 0u);
      ok = (i > 0 || mbar_wait_warp(kv_full(sk), (unsigned)(n / L::NQ) & 1u, abort_flag, nullptr, 82)) &&
           mbar_wait_warp(a_full(sa), (unsigned)(g / L::NA) & 1u, abort_flag, nullptr, 83);
      if (!ok) return;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (tc_elect()) {
        tt_mma_rows<D>(place(2 * g), kv_rows(), q_rows + stage(sa), idesc_s);
        tc_commit(full(2 * g));
      }
      __syncwarp();
      ++issued;
    };
    auto upstream = [&]() {  // dP of the tile whose S was issued last
      const int g = issued - 1, sb = g % L::NB;
      ok = mbar_wait_warp(b_full(sb), (unsigned)(g / L::NB) & 1u, abort_flag, nullptr, 85);
      if (!ok) return;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (tc_elect()) {
        tt_mma_rows<D>(place(2 * g + 1), kv_rows() + (unsigned long long)(TILE >> 4), do_rows + stage(sb), idesc_s);
        tc_commit(full(2 * g + 1));
        if (i + 1 == tiles) tc_commit(kv_empty(n % L::NQ));
      }
      __syncwarp();
    };
    scores();
    if (more && ok) upstream();
    if (NP == 3 && more && ok) scores();
    for (int g = 0; g < issued && ok; ++g) {
      const int sa = g % L::NA, sb = g % L::NB;
      const unsigned bit = 1u << (g & 3);
      const bool first = ends & bit << 4, last = ends & bit;
      ok = mbar_wait_warp(ready(2 * g), (unsigned)(2 * g / NP) & 1u, abort_flag, nullptr, 84);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (tc_elect()) tt_mma_weights<true>(tmem_dv, place(2 * g), do_cols + stage(sb), idesc_d, !first);
      __syncwarp();
      if (more) {
        if constexpr (NP == 3) upstream();
        else scores();
      }
      if (!ok) break;
      ok = mbar_wait_warp(ready(2 * g + 1), (unsigned)((2 * g + 1) / NP) & 1u, abort_flag, nullptr, 86);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (tc_elect()) {
        tt_mma_weights<true>(tmem_dk, place(2 * g + 1), q_cols + stage(sa), idesc_d, !first);
        tc_commit(a_empty(sa));
        tc_commit(b_empty(sb));  // (the statistics beside it have been read too)
        if (last) tc_commit(done);
      }
      __syncwarp();
      if (more) {
        if constexpr (NP == 3) scores();
        else upstream();
      }
    }
    if (!ok) {  // a bounded chance for the tensor pipe to finish before tensor memory is freed; the items' order goes on
      while (more) more = next.take(w++, lane) >= 0;
      if (tc_elect()) tc_commit(next.drained());
      __syncwarp();
      const unsigned long long limit = global_timer() + WAIT_LIMIT_NS;
      while (!mbar_try_wait(next.drained(), 0) && global_timer() < limit) {}
    }
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    const unsigned lanes = (unsigned)(q * 32) << 16;
    int g = 0, n = 0;
    bool ok = true;
    int block = next.take(0, lane);
    Item x = item(max(block, 0));
    for (int w = 1; block >= 0; ++w) {
      const int key = x.j0 + q * 32 + lane;
      const bool key_live = key < x.at.keys;
      for (int i = 0, t = 0; i < x.tiles && ok; ++i, ++g) {
        const int st = g % L::NB, r0 = x.lo + t * TT_B + half * 64;
        const unsigned tmem_s = place(2 * g), tmem_dp = place(2 * g + 1);
        t = t + 1 == x.each ? 0 : t + 1;
        // rows r0 + c that see this key: [c_lo, c_end)
        const int c_lo = a.span.causal ? key - a.span.first - r0 : 0;
        const long long pe = a.span.window > 0 ? (long long)key + a.span.window - a.span.first - r0 : 64;
        const int c_end = !key_live ? 0 : pe < 64 ? (int)max(pe, 0LL) : 64;
        const bool inside = __all_sync(0xffffffffu, c_lo <= 0 && c_end >= 64);
        ok = mbar_wait_warp(stat_full(st), (unsigned)(g / L::NB) & 1u, abort_flag, nullptr, 87) &&
             mbar_wait_warp(full(2 * g), (unsigned)(2 * g / NP) & 1u, abort_flag, nullptr, 88);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        float p[64];
        {
          unsigned(&u)[2][32] = reinterpret_cast<unsigned(&)[2][32]>(p);
          tc_ld32(tmem_s + lanes + (unsigned)(half * 64), u[0]);
          tc_ld32(tmem_s + lanes + (unsigned)(half * 64 + 32), u[1]);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        }
        const ulonglong2 *z = reinterpret_cast<const ulonglong2 *>(stat + st * 256 + half * 64);
        const unsigned long long f2 = tt_two(a.factor, a.factor);
#pragma unroll
        for (int j = 0; j < 64; j += 4) {
          const ulonglong2 v = z[j >> 2];
          const unsigned long long t = tt_exp2_two(tt_fma2(tt_two(p[j], p[j + 1]), f2, v.x));
          const unsigned long long u = tt_exp2_two(tt_fma2(tt_two(p[j + 2], p[j + 3]), f2, v.y));
          p[j] = tt_lo(t);
          p[j + 1] = tt_hi(t);
          p[j + 2] = tt_lo(u);
          p[j + 3] = tt_hi(u);
        }
        if (!inside) {
#pragma unroll
          for (int j = 0; j < 64; ++j)
            if (j < c_lo || j >= c_end) p[j] = 0.f;
          // What rows that see no key hold must not meet their weights of zero in dV and dK: this half's four warps clear them in both
          // tiles (S is done with q's; dP reads dout's meanwhile, into columns that count for nothing). Rows behind the last are
          // zeros already.
          const int keys = a.lengths ? max(0, min(a.seen, a.lengths[x.at.stream])) : a.seen, live = a.span.rows_end(a.n, keys);
          if (live < a.n && live < r0 + 64) {
            if (!(ok = mbar_wait_warp(b_full(st), (unsigned)(g / L::NB) & 1u, abort_flag, nullptr, 85))) break;
            const int from = max(live - r0, 0);
            for (int s = 0; s < SLABS; ++s)
              for (int e = from * 8 + q * 32 + lane; e < 64 * 8; e += 128) {
                const int to = s * TT_SLAB + half * 64 * 128 + e * 16;
                *reinterpret_cast<uint4 *>(base_ptr + (q_tile(g % L::NA) - base) + to) = make_uint4(0u, 0u, 0u, 0u);
                *reinterpret_cast<uint4 *>(base_ptr + (do_tile(st) - base) + to) = make_uint4(0u, 0u, 0u, 0u);
              }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
        }
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
          unsigned w[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) w[j] = tt_pack(p[c + 2 * j], p[c + 2 * j + 1]);
          tc_st16(tmem_s + lanes + (unsigned)(half * 64 + (c >> 1)), w);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(ready(2 * g));
        ok = mbar_wait_warp(full(2 * g + 1), (unsigned)((2 * g + 1) / NP) & 1u, abort_flag, nullptr, 89);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const ulonglong2 *de = reinterpret_cast<const ulonglong2 *>(stat + st * 256 + 128 + half * 64);
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
          unsigned u[32], w[16];
          tc_ld32(tmem_dp + lanes + (unsigned)(half * 64 + c), u);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const ulonglong2 v = de[(c + j) >> 2];
            const unsigned long long x = tt_mul2(tt_add2(tt_two(__uint_as_float(u[j]), __uint_as_float(u[j + 1])), v.x),
                                                 tt_two(p[c + j], p[c + j + 1]));
            const unsigned long long y = tt_mul2(tt_add2(tt_two(__uint_as_float(u[j + 2]), __uint_as_float(u[j + 3])), v.y),
                                                 tt_two(p[c + j + 2], p[c + j + 3]));
            w[j >> 1] = tt_pack(tt_lo(x), tt_hi(x));
            w[(j >> 1) + 1] = tt_pack(tt_lo(y), tt_hi(y));
          }
          if (!inside) {  // (a weight of zero has no part even where the other factor is not finite)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const int at_lo = c + 2 * j, at_hi = at_lo + 1;
              w[j] &= (at_lo < c_lo || at_lo >= c_end ? 0u : 0xffffu) | (at_hi < c_lo || at_hi >= c_end ? 0u : 0xffff0000u);
            }
          }
          tc_st16(tmem_dp + lanes + (unsigned)(half * 64 + (c >> 1)), w);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(ready(2 * g + 1));
      }
      const Item then = x;
      block = next.take(w, lane);
      if (block >= 0) x = item(block);
      if (ok) ok = mbar_wait_warp(done, (unsigned)n++ & 1u, abort_flag, nullptr, 90);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      ok = __all_sync(0xffffffffu, ok && !*abort_flag);
      const HeadView &o = half ? a.o2 : a.o1;  // one half of the warps stores dk, the other dv
      bf16 *row = reinterpret_cast<bf16 *>(o.p) + then.at.stream * o.s + (long long)key * o.r + then.at.head * o.h;
      tt_store_row(row, key < a.m, a, (half ? tmem_dv : tmem_dk) + lanes, 0, (a.dim + 15) & ~15, half ? 1.f : a.scale, false, ok);
    }
  }
  __syncwarp();
  pdl_launch_dependents();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

template <int D>
__global__ void __launch_bounds__(TT_BWD_THREADS, 1)
train_dq_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do,
                   const __grid_constant__ TtArgs a) {
  using L = TtBwd<D>;
  constexpr int SLABS = L::SLABS, TILE = L::TILE;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const unsigned base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char *base_ptr = smem_raw + (base - smem_u32(smem_raw));
  const unsigned bars = base + L::BAR_OFF;
  auto q_tile = [&](int s) { return base + (unsigned)(s * 2 * TILE); };  // and dout's behind it
  auto k_tile = [&](int s) { return base + (unsigned)(L::A_OFF + s * TILE); };
  auto v_tile = [&](int s) { return base + (unsigned)(L::B_OFF + s * TILE); };
  float *stat = reinterpret_cast<float *>(base_ptr + L::STAT_OFF);
  auto a_full = [&](int s) { return bars + 8u * s; };
  auto a_empty = [&](int s) { return bars + 32u + 8u * s; };
  auto b_full = [&](int s) { return bars + 64u + 8u * s; };
  auto b_empty = [&](int s) { return bars + 96u + 8u * s; };
  auto q_full = [&](int s) { return bars + 128u + 8u * s; };
  auto q_empty = [&](int s) { return bars + 144u + 8u * s; };
  auto dp_full = [&](int g) { return bars + 160u + 8u * (g & 1); };
  auto ds_ready = [&](int g) { return bars + 176u + 8u * (g & 1); };
  auto halves = [&](int q) { return bars + 192u + 8u * q; };  // of the two warps that share 32 rows
  const unsigned s_full = bars + 224, s_free = bars + 232, done = bars + 240;
  volatile unsigned *tmem_holder = reinterpret_cast<volatile unsigned *>(base_ptr + L::BAR_OFF + 248);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(base_ptr + L::BAR_OFF + 252);
  TtNext next{bars + 256u};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (unsigned bar : {s_full, dp_full(0), dp_full(1), done}) mbar_init(bar, 1);
    mbar_init(s_free, 8);
    mbar_init(ds_ready(0), 8);
    mbar_init(ds_ready(1), 8);
    for (int q = 0; q < 4; ++q) mbar_init(halves(q), 2);
    for (int s = 0; s < L::NQ; ++s) {
      mbar_init(q_full(s), 1);
      mbar_init(q_empty(s), 1);
    }
    for (int s = 0; s < L::NA; ++s) {
      mbar_init(a_full(s), 1);
      mbar_init(a_empty(s), 1);
    }
    for (int s = 0; s < L::NB; ++s) {
      mbar_init(b_full(s), 1);
      mbar_init(b_empty(s), 1);
    }
    next.init(9);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) tt_alloc(tmem_holder, 512u);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned tmem_s = *tmem_holder, tmem_dp0 = tmem_s + 128, tmem_dq = tmem_s + 384;
  pdl_wait();

  struct Item {
    TtPlace at;
    int r0, lo, tiles, ahead;  // ahead: tiles of a first pass, over the same keys
  };
  auto item = [&](int block) {
    Item x;
    x.at = tt_place(a, a.heads, a.span.causal != 0, 1, block);
    x.r0 = x.at.tile * TT_B;
    x.lo = a.span.lo(x.r0);
    const int end = a.span.end(min(x.r0 + TT_B, a.n) - 1, x.at.keys);
    x.tiles = end > x.lo ? (end - x.lo + TT_B - 1) / TT_B : 0;
    x.ahead = x.tiles == 2 && a.span.window > 0 && a.span.window <= TT_B ? 2 : 0;
    return x;
  };

  if (warp == 0) {
    int g = 0, n = 0, a_loads = 0, b_loads = 0;  // tiles of keys so far, items with any, loads issued
    bool ok = true;
    int block = (int)blockIdx.x;
    for (int w = 0;; ++w) {
      Item x = item(max(block, 0));
      while (block >= 0 && x.tiles == 0) {
        tt_store_zeros(a.o1, a, x.at, x.r0, a.n, lane);
        next.ask(lane);
        block = next.answer();
        x = item(max(block, 0));
      }
      next.push(w, block, lane);
      if (block < 0) break;
      bool asked = false;
      const int kh = x.at.head / a.share, sq = n % L::NQ;
      if (ok) {
        ok = mbar_wait_warp(q_empty(sq), ((unsigned)(n / L::NQ) & 1u) ^ 1u, abort_flag, nullptr, 91);
        if (ok && lane == 0) {
          mbar_expect_tx(q_full(sq), 2u * TILE);
          for (int s = 0; s < SLABS; ++s) {
            tma_load_4d(q_tile(sq) + s * TT_SLAB, &map_q, s * 64, x.at.head, x.r0, x.at.stream, q_full(sq));
            tma_load_4d(q_tile(sq) + TILE + s * TT_SLAB, &map_do, s * 64, x.at.head, x.r0, x.at.stream, q_full(sq));
          }
        }
        if (ok) ++n;
        __syncwarp();
      }
      const int jobs = x.ahead + x.tiles;
      for (int i = 0; i < jobs && ok; ++i, ++g) {
        const int sa = g % L::NA, sb = g % L::NB, j0 = x.lo + (i >= x.ahead ? i - x.ahead : i) * TT_B;
        ok = mbar_wait_warp(a_empty(sa), ((unsigned)(g / L::NA) & 1u) ^ 1u, abort_flag, nullptr, 91);
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(a_full(sa), (unsigned)TILE);
          for (int s = 0; s < SLABS; ++s) tma_load_4d(k_tile(sa) + s * TT_SLAB, &map_k, s * 64, kh, j0, x.at.stream, a_full(sa));
        }
        ++a_loads;
        __syncwarp();
        if (i + 1 == jobs) {
          next.ask(lane);
          asked = true;
        }
        ok = mbar_wait_warp(b_empty(sb), ((unsigned)(g / L::NB) & 1u) ^ 1u, abort_flag, nullptr, 91);
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(b_full(sb), (unsigned)TILE);
          for (int s = 0; s < SLABS; ++s) tma_load_4d(v_tile(sb) + s * TT_SLAB, &map_v, s * 64, kh, j0, x.at.stream, b_full(sb));
        }
        ++b_loads;
        __syncwarp();
      }
      if (!asked) next.ask(lane);
      block = next.answer();
    }
    if (*abort_flag) {  // copies in flight must land before the shared memory goes away
      const unsigned long long limit = global_timer() + WAIT_LIMIT_NS;
      for (int j = n > L::NQ ? n - L::NQ : 0; j < n; ++j)
        while (!mbar_try_wait(q_full(j % L::NQ), (unsigned)(j / L::NQ) & 1u) && global_timer() < limit) {}
      for (int j = a_loads > L::NA ? a_loads - L::NA : 0; j < a_loads; ++j)
        while (!mbar_try_wait(a_full(j % L::NA), (unsigned)(j / L::NA) & 1u) && global_timer() < limit) {}
      for (int j = b_loads > L::NB ? b_loads - L::NB : 0; j < b_loads; ++j)
        while (!mbar_try_wait(b_full(j % L::NB), (unsigned)(j / L::NB) & 1u) && global_timer() < limit) {}
    }
  } else if (warp == 1) {
    const int cols = (a.dim + 15) & ~15;
    const unsigned long long q_rows = tt_rows(q_tile(0)), k_rows = tt_rows(k_tile(0)), v_rows = tt_rows(v_tile(0)), k_cols = tt_cols(k_tile(0));
    auto stage = [](int s) { return (unsigned long long)(s * (TILE >> 4)); };
    const unsigned idesc_s = umma_idesc_bf16(TT_B), idesc_d = umma_idesc_bf16(cols) | UMMA_B_MN_MAJOR;
    // A tile of an item. S and dP are issued one tile ahead of dQ, into the next item too.
    struct Job {
      Item x;
      int i, g, n;  // tile of the item, of all; item
    };
    int w = 0;
    Job lead{};
    lead.i = lead.g = lead.n = -1;
    auto advance = [&]() {  // the next tile; false: none
      ++lead.g;
      if (++lead.i < lead.x.tiles + lead.x.ahead) return true;
      const int block = next.take(w++, lane);
      if (block < 0) return false;
      lead.x = item(block);
      lead.x.tiles = tt_uniform(lead.x.tiles);
      lead.x.ahead = tt_uniform(lead.x.ahead);
      lead.i = 0;
      ++lead.n;
      return true;
    };
    auto issue = [&](const Job &t) {
      const int sa = t.g % L::NA, sb = t.g % L::NB, sq = t.n % L::NQ;
      const unsigned long long q_at = q_rows + (unsigned long long)(sq * (2 * TILE >> 4));
      if (t.i == 0 && !mbar_wait_warp(q_full(sq), (unsigned)(t.n / L::NQ) & 1u, abort_flag, nullptr, 93)) return false;
      if (!mbar_wait_warp(a_full(sa), (unsigned)(t.g / L::NA) & 1u, abort_flag, nullptr, 92)) return false;
      // keys behind the stream's length must not meet the zeros of dS as anything but zeros
      const int have = t.x.at.keys - (t.x.lo + (t.i >= t.x.ahead ? t.i - t.x.ahead : t.i) * TT_B);
      if (have < TT_B && t.x.at.keys < a.m) tt_clear_rows(base_ptr + (k_tile(sa) - base), SLABS, have, lane);
      if (t.g > 0 && !mbar_wait_warp(s_free, (unsigned)(t.g - 1) & 1u, abort_flag, nullptr, 94)) return false;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (tc_elect()) {
        tt_mma_rows<D>(tmem_s, q_at, k_rows + stage(sa), idesc_s);
        tc_commit(s_full);
      }
      __syncwarp();
      if (!mbar_wait_warp(b_full(sb), (unsigned)(t.g / L::NB) & 1u, abort_flag, nullptr, 92)) return false;
      if (tc_elect()) {  // over dS of the tile before the last, whose product was issued before
        tt_mma_rows<D>(tmem_dp0 + (unsigned)((t.g & 1) * 128), q_at + (unsigned long long)(TILE >> 4), v_rows + stage(sb), idesc_s);
        tc_commit(dp_full(t.g));
        tc_commit(b_empty(sb));
        if (t.i + 1 == t.x.ahead + t.x.tiles) tc_commit(q_empty(sq));
      }
      __syncwarp();
      return true;
    };
    bool more = advance(), ok = !more || issue(lead);
    while (more && ok) {
      const Job now = lead;
      more = advance();
      ok = !more || issue(lead);
      if (!ok) break;
      ok = mbar_wait_warp(ds_ready(now.g), (unsigned)(now.g >> 1) & 1u, abort_flag, nullptr, 95);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (tc_elect()) {
        if (now.i >= now.x.ahead)
          tt_mma_weights<true>(tmem_dq, tmem_dp0 + (unsigned)((now.g & 1) * 128), k_cols + stage(now.g % L::NA), idesc_d, now.i > now.x.ahead);
        tc_commit(a_empty(now.g % L::NA));
        if (now.i + 1 == now.x.ahead + now.x.tiles) tc_commit(done);
      }
      __syncwarp();
    }
    if (!ok) {  // a bounded chance for the tensor pipe to finish before tensor memory is freed; the items' order goes on
      while (more) more = next.take(w++, lane) >= 0;
      if (tc_elect()) tc_commit(next.drained());
      __syncwarp();
      const unsigned long long limit = global_timer() + WAIT_LIMIT_NS;
      while (!mbar_try_wait(next.drained(), 0) && global_timer() < limit) {}
    }
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    const unsigned lanes = (unsigned)(q * 32) << 16;
    const int cols = (a.dim + 15) & ~15, mid = (cols / 2 + 15) & ~15;  // each half of the warps stores half of the columns
    int g = 0, n = 0, exact = 0;
    bool ok = true;
    // dout . out is off by what out was rounded by, which counts in rows of few keys (a window of 12: dq and dk half again as far from
    // 64 bits as their own rounding leaves them). Where all of a row's keys lie in this one tile, the same sum over keys, p dP, is
    // at hand in 32 bits; under a narrow window, whose keys lie in two, a first pass over both takes it. (The kernel of dk and dv
    // then finds it in place of the other.)
    auto exact_part = [&](const float (&p)[64], unsigned tmem_dp, int c_lo, int c_end) {
      float t = 0.f;
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        unsigned u[32];
        tc_ld32(tmem_dp + lanes + (unsigned)(half * 64 + c), u);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (c + j >= c_lo && c + j < c_end) t = fmaf(p[c + j], __uint_as_float(u[j]), t);
      }
      return t;
    };
    auto exact_delta = [&](float part) {
      // (of two places in turn: the other half has read this one's before it arrives for the next)
      float *both = stat + (exact & 1) * 256 + q * 32 + lane;
      both[half * 128] = part;
      __syncwarp();
      if (lane == 0) mbar_arrive(halves(q));
      const bool met = mbar_wait_warp(halves(q), (unsigned)exact & 1u, abort_flag, nullptr, 99);
      ++exact;
      return met ? both[0] + both[128] : NAN;
    };
    int block = next.take(0, lane);
    Item x = item(max(block, 0));
    auto statistics = [&](float &z, float &delta) {
      const int row = x.r0 + q * 32 + lane;
      const long long at = ((long long)x.at.stream * a.heads + x.at.head) * a.n + row;
      z = row < a.n ? a.lse[at] : -INFINITY;
      delta = row < a.n ? a.delta[at] : 0.f;
    };
    float z, delta;
    statistics(z, delta);
    for (int w = 1; block >= 0; ++w) {
      const int row = x.r0 + q * 32 + lane;
      const int row_lo = a.span.lo(row), row_end = a.span.end(row, x.at.keys);
      const int warp_lo = a.span.lo(x.r0 + q * 32 + 31), warp_end = a.span.end(x.r0 + q * 32, x.at.keys);
      const float lse = z == -INFINITY ? -INFINITY : -(z * TT_LOG2E);  // to add; a row that sees no key has no weights: 2^(s - infinity)
      float part = 0.f;
      for (int i = -x.ahead; i < x.tiles && ok; ++i, ++g) {
        const int j0 = x.lo + (i < 0 ? i + x.ahead : i) * TT_B + half * 64;
        const unsigned tmem_dp = tmem_dp0 + (unsigned)((g & 1) * 128);
        const int c_lo = row_lo - j0, c_end = row_end - j0;
        const bool inside = warp_lo <= j0 && warp_end >= j0 + 64;
        ok = mbar_wait_warp(s_full, (unsigned)g & 1u, abort_flag, nullptr, 96);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        float p[64];
        {
          unsigned(&u)[2][32] = reinterpret_cast<unsigned(&)[2][32]>(p);
          tc_ld32(tmem_s + lanes + (unsigned)(half * 64), u[0]);
          tc_ld32(tmem_s + lanes + (unsigned)(half * 64 + 32), u[1]);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(s_free);
        const unsigned long long f2 = tt_two(a.factor, a.factor), z2 = tt_two(lse, lse);
#pragma unroll
        for (int j = 0; j < 64; j += 2) {
          const unsigned long long t = tt_exp2_two(tt_fma2(tt_two(p[j], p[j + 1]), f2, z2));
          p[j] = tt_lo(t);
          p[j + 1] = tt_hi(t);
        }
        ok = mbar_wait_warp(dp_full(g), (unsigned)(g >> 1) & 1u, abort_flag, nullptr, 97);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (!inside) {
#pragma unroll
          for (int j = 0; j < 64; ++j)
            if (j < c_lo || j >= c_end) p[j] = 0.f;
        }
        if (i < 0 || x.tiles == 1) {
          part += exact_part(p, tmem_dp, c_lo, c_end);
          if (i == -1 || x.tiles == 1) {
            delta = exact_delta(part);
            if (half == 0 && row < a.n) a.delta[((long long)x.at.stream * a.heads + x.at.head) * a.n + row] = delta;
          }
        }
        if (i < 0) {
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(ds_ready(g));
          continue;
        }
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
          unsigned u[32], v[16];
          tc_ld32(tmem_dp + lanes + (unsigned)(half * 64 + c), u);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          const unsigned long long d2 = tt_two(-delta, -delta);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const unsigned long long y = tt_mul2(tt_add2(tt_two(__uint_as_float(u[j]), __uint_as_float(u[j + 1])), d2),
                                                 tt_two(p[c + j], p[c + j + 1]));
            p[c + j] = tt_lo(y);
            p[c + j + 1] = tt_hi(y);
          }
          if (!inside) {  // (a weight of zero has no part even where the other factor is not finite)
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c + j < c_lo || c + j >= c_end) p[c + j] = 0.f;
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = tt_pack(p[c + 2 * j], p[c + 2 * j + 1]);
          tc_st16(tmem_dp + lanes + (unsigned)(half * 64 + (c >> 1)), v);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_ready(g));
      }
      // the next item's statistics are on their way while this one's rows are stored
      const Item then = x;
      block = next.take(w, lane);
      if (block >= 0) {
        x = item(block);
        statistics(z, delta);
      }
      if (ok) ok = mbar_wait_warp(done, (unsigned)n++ & 1u, abort_flag, nullptr, 98);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      bf16 *o = reinterpret_cast<bf16 *>(a.o1.p) + then.at.stream * a.o1.s + (long long)row * a.o1.r + then.at.head * a.o1.h;
      ok = __all_sync(0xffffffffu, ok && !*abort_flag);
      tt_store_row(o, row < a.n, a, tmem_dq + lanes, half ? mid : 0, half ? cols : mid, a.scale, false, ok);
    }
  }
  __syncwarp();
  pdl_launch_dependents();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_s), "r"(512u));
  }
}

// Whether TMA can address the rows: contiguous columns, 16-byte boundaries, strides that are no repetition.
bool tt_addressable(const HeadView &x, long long streams, long long rows, long long heads) {
  auto stride = [](long long s, long long extent) { return extent <= 1 || (s > 0 && s % 8 == 0 && s < (1ll << 38)); };
  return x.c == 1 && reinterpret_cast<uintptr_t>(x.p) % 16 == 0 && stride(x.s, streams) && stride(x.r, rows) && stride(x.h, heads);
}

CUtensorMap tt_map(const HeadView &x, long long streams, long long rows, long long heads, int dim) {
  CUtensorMap map;
  auto bytes = [](long long s, long long extent) { return extent <= 1 ? 16ull : (unsigned long long)s * 2; };
  const unsigned long long extent[4] = {(unsigned long long)dim, (unsigned long long)heads, (unsigned long long)rows,
                                        (unsigned long long)streams};
  const unsigned long long strides[3] = {bytes(x.h, heads), bytes(x.r, rows), bytes(x.s, streams)};
  tc_make_map_heads(&map, x.p, extent, strides, TT_B);
  return map;
}

bool tt_rows16(const HeadView &x) {
  return x.c == 1 && reinterpret_cast<uintptr_t>(x.p) % 16 == 0 && x.s % 8 == 0 && x.r % 8 == 0 && x.h % 8 == 0;
}

template <int D>
void forward(const TrainAttention &a, cudaStream_t st) {
  TtArgs t = tt_args(a, a.n);
  t.o1 = a.out;
  t.q = a.q;
  t.k = a.k;
  t.v = a.v;
  t.vec = tt_rows16(a.out);
  const size_t smem = 3 * (size_t)(D / 64) * TT_SLAB + 128 + 1024;
  static SharedMemoryOnce once;
  once.set(train_forward_tc_kernel<D>, (int)smem);
  train_forward_tc_kernel<D><<<tt_grid(t, a.heads), TT_FWD_THREADS, smem, st>>>(
      tt_map(a.q, a.streams, a.n, a.heads, a.dim), tt_map(a.k, a.streams, a.m, a.groups, a.dim),
      tt_map(a.v, a.streams, a.m, a.groups, a.dim), t);
  LB_LAUNCH_CHECK();
}

void forward_pair(const TrainAttention &a, cudaStream_t st) {
  TtArgs t = tt_args(a, a.n);
  t.tiles = (a.n + 2 * TT_B - 1) / (2 * TT_B);
  t.o1 = a.out;
  t.q = a.q;
  t.k = a.k;
  t.v = a.v;
  t.vec = tt_rows16(a.out);
  static SharedMemoryOnce once;
  once.set(train_forward_pair_kernel, TT_PAIR_SMEM);
  train_forward_pair_kernel<<<tt_grid(t, a.heads), TT_BWD_THREADS, TT_PAIR_SMEM, st>>>(
      tt_map(a.q, a.streams, a.n, a.heads, a.dim), tt_map(a.k, a.streams, a.m, a.groups, a.dim),
      tt_map(a.v, a.streams, a.m, a.groups, a.dim), t);
  LB_LAUNCH_CHECK();
}

template <int D>
void backward(const TrainAttention &a, float *delta, cudaStream_t st) {
  const CUtensorMap mq = tt_map(a.q, a.streams, a.n, a.heads, a.dim), mk = tt_map(a.k, a.streams, a.m, a.groups, a.dim),
                    mv = tt_map(a.v, a.streams, a.m, a.groups, a.dim), md = tt_map(a.dout, a.streams, a.n, a.heads, a.dim);
  constexpr int smem = TtBwd<D>::TOTAL;
  TtArgs t = tt_args(a, a.n);
  t.delta = delta;
  t.o1 = a.dq;
  t.vec = tt_rows16(a.dq);
  static SharedMemoryOnce once_dq;
  once_dq.set(train_dq_tc_kernel<D>, smem);
  launch_pdl(train_dq_tc_kernel<D>, dim3(tt_grid(t, a.heads)), dim3(TT_BWD_THREADS), (size_t)smem, st, true, mq, mk, mv, md, t);
  t = tt_args(a, a.m);
  t.delta = delta;
  t.o1 = a.dk;
  t.o2 = a.dv;
  t.vec = tt_rows16(a.dk) && tt_rows16(a.dv);
  static SharedMemoryOnce once_dkv;
  once_dkv.set(train_dkv_tc_kernel<D>, smem);
  launch_pdl(train_dkv_tc_kernel<D>, dim3(tt_grid(t, a.groups)), dim3(TT_BWD_THREADS), (size_t)smem, st, true, mq, mk, mv, md, t);
}

}  // namespace

bool train_attention_tc_supports(const TrainAttention &a, bool backward) {
  if (!a.bf16 || a.dim % 8 != 0) return false;
  const long long s = a.streams;
  return tt_addressable(a.q, s, a.n, a.heads) && tt_addressable(a.k, s, a.m, a.groups) && tt_addressable(a.v, s, a.m, a.groups) &&
         (backward ? tt_addressable(a.dout, s, a.n, a.heads) && a.dq.c == 1 && a.dk.c == 1 && a.dv.c == 1 : a.out.c == 1);
}

void launch_train_attention_forward_tc(const TrainAttention &a, cudaStream_t st) {
  // Two tiles per CTA: 4 streams of 2048 rows of 16 heads 82 -> 70 us, 8192 rows 227 -> 210, 64 streams of 300 rows of 8 heads 54 -> 47,
  // 129 rows no difference. Rows that see few keys, by a window, leave little to alternate with.
  const int seen = a.window > 0 && a.window < a.m ? a.window : a.m;
  if (a.dim <= 64 && min(a.n, seen) > TT_B) forward_pair(a, st);
  else if (a.dim <= 64) forward<64>(a, st);
  else forward<128>(a, st);
}

void launch_train_attention_backward_tc(const TrainAttention &a, float *delta, cudaStream_t st) {
  if (a.dim <= 64) backward<64>(a, delta, st);
  else backward<128>(a, delta, st);
}

}  // namespace lb

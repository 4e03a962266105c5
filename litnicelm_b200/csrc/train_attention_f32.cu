// Attention with its backward pass for training in 32 bits on the sm_100a tensor cores. The mathematics is that of train_attention.cu, the
// division of work that of train_attention_tc.cu.
//
// Operands are in three bfloat16 parts, x = x0 + x1 + x2, each the part before it left over: all 24 bits of a finite x. A product
// is the six of parts whose terms count, smallest first: (0,2) (2,0) (1,1) (0,1) (1,0) (0,0); what is left out is below 2^-23 of a
// term. The tensor pipe truncates when it adds, so an accumulator in tensor memory holds one tile's product and is added to a
// sum in registers, rounded to nearest. Queries, keys, values and upstream gradients are split once by a kernel in front
// (which also clears keys behind a stream's length or every row, and rows that see no key, and sums dout . out), weights and their gradients in registers on their way
// to tensor memory: of the 128 columns that a tile's scores took, each half of the warps writes the first two parts over its own
// 64, and the third behind them.
//
// Heads of more than 64 dimensions (H = 2): a tile's parts are 96 KB, and two tiles of products do not fit beside two resident ones. A
// CTA then makes 64 of the result's dimensions, and its products' operands come in units of 64 dimensions through four places of shared
// memory, all four together where a sum runs over all dimensions (small parts first there too).
//
// Bound: at the sizes that such models train at, latency: 8 streams of 250 rows, 8 heads of 64 take 67 us forward and backward (split 2 x 9,
// forward 13, backward 35 us) with 128 CTAs a result of dependent stages of six products each; with 32-bit products on the FMA
// pipe it was 219 us. 2000 rows of 8 heads of 128: 419 us, 1957 that way; the six products are 100 us of it at the pipe's rate.
//
// A CTA: warp 0 issues TMA, warp 1 owns tensor memory and issues the MMAs, eight warps (a thread: a row or key, half of the
// tile's columns, half of the dimensions of a sum; with both sums and the parts in the making dk and dv's spill 500 bytes at H = 1, 372
// at H = 2). Every wait is bounded; one that runs out ends the CTA, whose results are then NaN.
#include "train_attention_tc.cuh"

namespace lb {

namespace {

constexpr int TF_THREADS = 320, TF_PART = TT_SLAB, TF_TILE = 3 * TF_PART;

// ---- operands in parts --------------------------------------------------------------------------------------------------------

struct TfTensor {
  HeadView x;
  int rows, heads, keys;  // keys: rows behind a stream's length are cleared; else rows that see no key
  bf16 *part;             // [3][streams][heads][rows][64 H]
  int blocks, vec;
};
struct TfSplit {
  TfTensor t[4];
  int count, streams, dim, chunks;  // chunks: of eight elements, 8 H to a row
  int seen;
  TrainSpan span;
  const int *lengths;
  HeadView out;           // with delta: of the last tensor, dout
  float *delta;
};

__device__ __forceinline__ float tf_in_range(float x) {
  const float top = 3.3895313892515355e38f;  // (2 - 2^-7) 2^127, the largest bfloat16
  return fabsf(x) > top && fabsf(x) < INFINITY ? copysignf(top, x) : x;
}

__global__ void __launch_bounds__(256) train_split_kernel(const __grid_constant__ TfSplit g) {
  pdl_launch_dependents();
  int b = (int)blockIdx.x, which = 0;
  while (which + 1 < g.count && b >= g.t[which].blocks) b -= g.t[which++].blocks;
  const TfTensor &t = g.t[which];
  const int each_block = 256 / g.chunks, per = (t.rows + each_block - 1) / each_block;
  const int head_at = b / per, s = head_at / t.heads, h = head_at - s * t.heads;
  const int row = (b - head_at * per) * each_block + (int)threadIdx.x / g.chunks, c = (int)threadIdx.x % g.chunks * 8;
  const bool in = row < t.rows;
  const int keys = g.lengths ? max(0, min(g.seen, g.lengths[s])) : g.seen, live = t.keys ? keys : g.span.rows_end(t.rows, keys);
  float x[8] = {};
  const long long off = (long long)s * t.x.s + (long long)row * t.x.r + (long long)h * t.x.h + (long long)c * t.x.c;
  if (row < live) {
    const float *p = reinterpret_cast<const float *>(t.x.p) + off;
    if (t.vec && c + 8 <= g.dim) {
      const float4 u = *reinterpret_cast<const float4 *>(p), v = *reinterpret_cast<const float4 *>(p + 4);
      x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
      x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < g.dim) x[j] = p[j * t.x.c];
    }
  }
  if (in) {
    unsigned w[3][4];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      float a = x[j], e = x[j + 1];
#pragma unroll
      for (int q = 0; q < 3; ++q) {
        // (the first part of a finite element is finite: the last 2^119 below the largest would round to infinity)
        const __nv_bfloat162 v = q ? __floats2bfloat162_rn(a, e) : __floats2bfloat162_rn(tf_in_range(a), tf_in_range(e));
        w[q][j >> 1] = *reinterpret_cast<const unsigned *>(&v);
        const float2 f = __bfloat1622float2(v);
        a -= f.x;
        e -= f.y;
      }
    }
    const long long ld = g.chunks * 8, each = (long long)g.streams * t.heads * t.rows * ld, to = ((long long)head_at * t.rows + row) * ld + c;
#pragma unroll
    for (int q = 0; q < 3; ++q) *reinterpret_cast<uint4 *>(t.part + q * each + to) = make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]);
  }
  if (g.delta && which == g.count - 1) {
    float d = 0.f;
    if (in) {
      const float *o = reinterpret_cast<const float *>(g.out.p) + (long long)s * g.out.s + (long long)row * g.out.r +
                       (long long)h * g.out.h + (long long)c * g.out.c;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < g.dim) d = fmaf(x[j], o[j * g.out.c], d);
    }
    for (int o = g.chunks / 2; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (in && c == 0) g.delta[(long long)head_at * t.rows + row] = d;
  }
}

// ---- helpers of the three kernels ----------------------------------------------------------------------------------------------

// The product of rows of a and rows of b over 64 dimensions, smallest parts first. (Descriptors differ by constants: see tt_mma_rows in
// train_attention_tc.cu.)
__device__ __forceinline__ void tf_mma_rows(unsigned d, unsigned a, unsigned b, unsigned idesc) {
  const unsigned long long da = umma_desc_k128(a), db = umma_desc_k128(b);
#pragma unroll
  for (int p = 0; p < 6; ++p) {
    const int pa = p == 0 ? 0 : p == 1 ? 2 : p == 2 ? 1 : p == 3 ? 0 : p == 4 ? 1 : 0;
    const int pb = p == 0 ? 2 : p == 1 ? 0 : p == 2 ? 1 : p == 3 ? 1 : p == 4 ? 0 : 0;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
      tc_mma_f16(d, da + (unsigned long long)(pa * (TF_PART >> 4) + ks * 2), db + (unsigned long long)(pb * (TF_PART >> 4) + ks * 2), idesc,
                 (p | ks) ? 1u : 0u);
  }
}
// Weights in tensor memory (parts where tf_store_parts puts them) by rows of b.
__device__ __forceinline__ void tf_mma_weights(unsigned d, unsigned w, unsigned b, unsigned idesc) {
  const unsigned long long db = umma_desc_mn128(b, TT_SLAB);
#pragma unroll
  for (int p = 0; p < 6; ++p) {
    const int pa = p == 0 ? 0 : p == 1 ? 2 : p == 2 ? 1 : p == 3 ? 0 : p == 4 ? 1 : 0;
    const int pb = p == 0 ? 2 : p == 1 ? 0 : p == 2 ? 1 : p == 3 ? 1 : p == 4 ? 0 : 0;
#pragma unroll
    for (int ks = 0; ks < TT_B / 16; ++ks) {
      const unsigned at = pa == 2 ? 128u + (unsigned)(ks * 8) : (unsigned)((ks >> 2) * 64 + pa * 32 + (ks & 3) * 8);
      tc_mma_f16_ts(d, w + at, db + (unsigned long long)((pb * TF_PART + ks * 16 * 128) >> 4), idesc, (p | ks) ? 1u : 0u);
    }
  }
}
// 32 weights of this thread's row, columns c .. c + 31 of its half, as parts.
__device__ __forceinline__ void tf_store_parts(unsigned w, int half, int c, const float *x) {
  unsigned part[3][16];
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    float a = x[j], e = x[j + 1];
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(a, e);
      part[q][j >> 1] = *reinterpret_cast<const unsigned *>(&v);
      const float2 f = __bfloat1622float2(v);
      a -= f.x;
      e -= f.y;
    }
  }
  tc_st16(w + (unsigned)(half * 64 + (c >> 1)), part[0]);
  tc_st16(w + (unsigned)(half * 64 + 32 + (c >> 1)), part[1]);
  tc_st16(w + (unsigned)(128 + half * 32 + (c >> 1)), part[2]);
}
// A finished tile's 32 columns of this thread added to its sums.
__device__ __forceinline__ void tf_add(unsigned at, float keep, float (&sum)[32]) {
  unsigned r[32];
  tc_ld32(at, r);
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int j = 0; j < 32; ++j) sum[j] = fmaf(sum[j], keep, __uint_as_float(r[j]));
}
__device__ __forceinline__ void tf_store_sums(const HeadView &o, long long off, const TtArgs &a, int c0, const float (&sum)[32], float f) {
  float *row = reinterpret_cast<float *>(o.p) + off;
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    if (a.vec && c0 + j + 4 <= a.dim) {
      *reinterpret_cast<float4 *>(row + c0 + j) = make_float4(sum[j] * f, sum[j + 1] * f, sum[j + 2] * f, sum[j + 3] * f);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c0 + j + e < a.dim) row[(long long)(c0 + j + e) * o.c] = sum[j + e] * f;
    }
  }
}
// Three parts of 128 rows of head `at` (of `each` heads in all).
__device__ __forceinline__ void tf_load(unsigned to, const CUtensorMap *map, int row, int at, int each, unsigned bar, int x = 0) {
#pragma unroll
  for (int p = 0; p < 3; ++p) tma_load_4d(to + p * TF_PART, map, x, 0, row, p * each + at, bar);
}

// Units of 64 dimensions through four places of shared memory (H = 2): the producer's and the consumer's count of units. Barriers:
// full of place s at bars + 8 s, empty at bars + 32 + 8 s.
struct TfRing {
  unsigned base, bars;
  int at = 0;
  __device__ unsigned place(int u) const { return base + (unsigned)((u & 3) * TF_TILE); }
  __device__ unsigned full(int u) const { return bars + 8u * (u & 3); }
  __device__ unsigned empty(int u) const { return bars + 32u + 8u * (u & 3); }
};
__device__ __forceinline__ bool tf_put(TfRing &r, const CUtensorMap *map, int x, int row, int head, int each, int lane,
                                       volatile int *abort_flag) {
  if (!mbar_wait_warp(r.empty(r.at), ((unsigned)(r.at >> 2) & 1u) ^ 1u, abort_flag, nullptr, 142)) return false;
  if (lane == 0) {
    mbar_expect_tx(r.full(r.at), TF_TILE);
    tf_load(r.place(r.at), map, row, head, each, r.full(r.at), x);
  }
  __syncwarp();
  ++r.at;
  return true;
}
__device__ __forceinline__ bool tf_take(const TfRing &r, int u, volatile int *abort_flag) {
  return mbar_wait_warp(r.full(u), (unsigned)(u >> 2) & 1u, abort_flag, nullptr, 143);
}
__device__ __forceinline__ void tf_drain(const TfRing &r) {  // copies in flight land before the shared memory goes away
  const unsigned long long limit = global_timer() + WAIT_LIMIT_NS;
  for (int u = r.at > 4 ? r.at - 4 : 0; u < r.at; ++u)
    while (!mbar_try_wait(r.full(u), (unsigned)(u >> 2) & 1u) && global_timer() < limit) {}
}
// Four units a0 b0 a1 b1 from the ring's next places: d = a . b over 128 dimensions. Issued and given back.
__device__ __forceinline__ bool tf_mma_ring(TfRing &r, unsigned d, unsigned idesc, unsigned done, volatile int *abort_flag) {
  for (int u = 0; u < 4; ++u)
    if (!tf_take(r, r.at + u, abort_flag)) return false;
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (tc_elect()) {
    // units in order of place: a0, b0, a1, b1 start at any of the four
    const unsigned a0 = r.place(r.at), b0 = r.place(r.at + 1), a1 = r.place(r.at + 2), b1 = r.place(r.at + 3);
    const unsigned long long da[2] = {umma_desc_k128(a0), umma_desc_k128(a1)}, db[2] = {umma_desc_k128(b0), umma_desc_k128(b1)};
#pragma unroll
    for (int p = 0; p < 6; ++p) {
      const int pa = p == 0 ? 0 : p == 1 ? 2 : p == 2 ? 1 : p == 3 ? 0 : p == 4 ? 1 : 0;
      const int pb = p == 0 ? 2 : p == 1 ? 0 : p == 2 ? 1 : p == 3 ? 1 : p == 4 ? 0 : 0;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          tc_mma_f16(d, da[h] + (unsigned long long)(pa * (TF_PART >> 4) + ks * 2), db[h] + (unsigned long long)(pb * (TF_PART >> 4) + ks * 2),
                     idesc, (p | h | ks) ? 1u : 0u);
    }
    for (int u = 0; u < 4; ++u) tc_commit(r.empty(r.at + u));
    tc_commit(done);
  }
  __syncwarp();
  r.at += 4;
  return true;
}
// One unit: d = weights . its rows.
__device__ __forceinline__ bool tf_mma_ring_weights(TfRing &r, unsigned d, unsigned w, unsigned idesc, unsigned done, volatile int *abort_flag) {
  if (!tf_take(r, r.at, abort_flag)) return false;
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (tc_elect()) {
    tf_mma_weights(d, w, r.place(r.at), idesc);
    tc_commit(r.empty(r.at));
    tc_commit(done);
  }
  __syncwarp();
  ++r.at;
  return true;
}

#define TF_WAIT(bar, parity, where) mbar_wait_warp(bar, (unsigned)(parity) & 1u, abort_flag, nullptr, where)
#define TF_AFTER() asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory")
#define TF_READY(bar)                                                       \
  do {                                                                      \
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");            \
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");        \
    __syncwarp();                                                           \
    if (lane == 0) mbar_arrive(bar);                                        \
  } while (0)

constexpr int TF_STAT_OFF = 4 * TF_TILE, TF_BAR_OFF = TF_STAT_OFF + 4 * 128 * 4, TF_SMEM = TF_BAR_OFF + 256 + 1024;
static_assert(TF_SMEM <= 227 * 1024, "");

// ---- forward --------------------------------------------------------------------------------------------------------------------

template <int H>
__global__ void __launch_bounds__(TF_THREADS, 1)
train_forward_f32_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TtArgs a) {
  extern __shared__ unsigned char smem_raw[];
  const unsigned base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char *base_ptr = smem_raw + (base - smem_u32(smem_raw));
  const unsigned q_off = base, k_off = base + TF_TILE, v_off = base + 2 * TF_TILE, bars = base + TF_BAR_OFF;
  float *stat = reinterpret_cast<float *>(base_ptr + TF_STAT_OFF);
  const unsigned q_full = bars + 64, k_full = bars + 72, v_full = bars + 80, s_full = bars + 88, p_ready = bars + 96, o_full = bars + 104;
  auto halves = [&](int q) { return bars + 112u + 8u * q; };  // of the two warps that share 32 rows
  volatile unsigned *tmem_holder = reinterpret_cast<volatile unsigned *>(base_ptr + TF_BAR_OFF + 240);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(base_ptr + TF_BAR_OFF + 244);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int oh = H == 2 ? (int)blockIdx.x & 1 : 0;  // which 64 dimensions of the result
  const TtPlace at = tt_place(a, a.heads, a.span.causal != 0, H);
  const int r0 = at.tile * TT_B, r1 = min(r0 + TT_B, a.n), kh = at.head / a.share;
  const int lo = a.span.lo(r0), end = a.span.end(r1 - 1, at.keys);
  const int tiles = end > lo ? (end - lo + TT_B - 1) / TT_B : 0;

  if (threadIdx.x == 0) {
    for (unsigned bar : {q_full, k_full, v_full, s_full, o_full}) mbar_init(bar, 1);
    mbar_init(p_ready, 8);
    for (int q = 0; q < 4; ++q) mbar_init(halves(q), 2);
    if (H == 2)
      for (int i = 0; i < 8; ++i) mbar_init(bars + 8u * i, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) tt_alloc(tmem_holder, 256u);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  TF_AFTER();
  const unsigned tmem_s = *tmem_holder, tmem_o = tmem_s + 192;
  pdl_wait();

  if (warp == 0) {
    if constexpr (H == 2) {
      TfRing ring{base, bars};
      const int query_head = at.stream * a.heads + at.head, key_head = at.stream * a.groups + kh;
      const int queries = a.streams * a.heads, keys = a.streams * a.groups;
      bool ok = true;
      for (int i = 0; i < tiles && ok; ++i) {
        const int j0 = lo + i * TT_B;
        for (int d = 0; d < 2 && ok; ++d)
          ok = tf_put(ring, &map_q, d * 64, r0, query_head, queries, lane, abort_flag) &&
               tf_put(ring, &map_k, d * 64, j0, key_head, keys, lane, abort_flag);
        ok = ok && tf_put(ring, &map_v, oh * 64, j0, key_head, keys, lane, abort_flag);
      }
      if (*abort_flag) tf_drain(ring);
    } else {
    int k_loads = 0, v_loads = 0;
    bool ok = true;
    if (lane == 0 && tiles > 0) {
      mbar_expect_tx(q_full, TF_TILE);
      tf_load(q_off, &map_q, r0, at.stream * a.heads + at.head, a.streams * a.heads, q_full);
    }
    for (int i = 0; i < tiles && ok; ++i) {
      const int j0 = lo + i * TT_B, key_head = at.stream * a.groups + kh;
      if (i > 0) ok = TF_WAIT(s_full, i - 1, 101);  // the scores have read the keys
      if (!ok) break;
      if (lane == 0) {
        mbar_expect_tx(k_full, TF_TILE);
        tf_load(k_off, &map_k, j0, key_head, a.streams * a.groups, k_full);
      }
      ++k_loads;
      if (i > 0) ok = TF_WAIT(o_full, i - 1, 102);  // P V has read the values
      if (!ok) break;
      if (lane == 0) {
        mbar_expect_tx(v_full, TF_TILE);
        tf_load(v_off, &map_v, j0, key_head, a.streams * a.groups, v_full);
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
    }
  } else if (warp == 1) {
    const int cols = H == 2 ? 64 : (a.dim + 15) & ~15;
    const unsigned idesc_s = umma_idesc_bf16(TT_B), idesc_o = umma_idesc_bf16(cols) | UMMA_B_MN_MAJOR;
    bool ok = H == 2 || tiles == 0 ? true : TF_WAIT(q_full, 0, 103);
    int i = 0;
    TfRing ring{base, bars};
    for (; i < tiles && ok; ++i) {
      if constexpr (H == 2) {
        ok = tf_mma_ring(ring, tmem_s, idesc_s, s_full, abort_flag) && TF_WAIT(p_ready, i, 106) &&
             tf_mma_ring_weights(ring, tmem_o, tmem_s, idesc_o, o_full, abort_flag);
        continue;
      }
      ok = TF_WAIT(k_full, i, 104);
      if (!ok) break;
      TF_AFTER();
      if (tc_elect()) {
        tf_mma_rows(tmem_s, q_off, k_off, idesc_s);
        tc_commit(s_full);
      }
      __syncwarp();
      ok = TF_WAIT(v_full, i, 105) && TF_WAIT(p_ready, i, 106);
      if (!ok) break;
      TF_AFTER();
      if (tc_elect()) {
        tf_mma_weights(tmem_o, tmem_s, v_off, idesc_o);
        tc_commit(o_full);
      }
      __syncwarp();
    }
    if (!ok) {  // a bounded chance for the tensor pipe to finish before tensor memory is freed
      if (tc_elect()) tc_commit(o_full);
      __syncwarp();
      const unsigned long long limit = global_timer() + WAIT_LIMIT_NS;
      while (!mbar_try_wait(o_full, (unsigned)i & 1u) && global_timer() < limit) {}
    }
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    const unsigned lanes = (unsigned)(q * 32) << 16;
    const int r = q * 32 + lane, row = r0 + r;
    const int row_lo = a.span.lo(row), row_end = a.span.end(row, at.keys);
    const int warp_lo = a.span.lo(r0 + q * 32 + 31), warp_end = a.span.end(r0 + q * 32, at.keys);
    float m = TT_NEG, l = 0.f, sum[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) sum[j] = 0.f;
    bool ok = true;
    for (int i = 0; i < tiles && ok; ++i) {
      const int j0 = lo + i * TT_B + half * 64;
      const int c_lo = row_lo - j0, c_end = row_end - j0;  // keys j0 + c that this row sees
      const bool inside = warp_lo <= j0 && warp_end >= j0 + 64;
      ok = TF_WAIT(s_full, i, 107);
      if (!ok) break;
      TF_AFTER();
      float s[64];
      {
        unsigned(&u)[2][32] = reinterpret_cast<unsigned(&)[2][32]>(s);
        tc_ld32(tmem_s + lanes + (unsigned)(half * 64), u[0]);
        tc_ld32(tmem_s + lanes + (unsigned)(half * 64 + 32), u[1]);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      }
#pragma unroll
      for (int j = 0; j < 64; ++j) s[j] = __fmul_rn(s[j], a.factor);  // (rounded, or the difference from m is not)
      if (!inside) {
#pragma unroll
        for (int j = 0; j < 64; ++j)
          if (j >= c_end || j < c_lo) s[j] = -INFINITY;  // weight zero against any reference
      }
      float mq[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int j = 4; j < 64; ++j) mq[j & 3] = fmaxf(mq[j & 3], s[j]);
      // the row's maximum over both halves
      float *both = stat + (i & 1) * 256 + r;
      both[half * 128] = fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3]));
      __syncwarp();
      if (lane == 0) mbar_arrive(halves(q));
      ok = TF_WAIT(halves(q), i, 109);
      if (!ok) break;
      const float mx = fmaxf(m, fmaxf(both[0], both[128]));
      const float keep = tt_exp2(m - mx);
      m = mx;
      l *= keep;
      float lq[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 64; ++j) {
        s[j] = tt_exp2(s[j] - m);
        lq[j & 3] += s[j];
      }
      l += (lq[0] + lq[1]) + (lq[2] + lq[3]);
      tf_store_parts(tmem_s + lanes, half, 0, s);
      tf_store_parts(tmem_s + lanes, half, 32, s + 32);
      TF_READY(p_ready);
      ok = TF_WAIT(o_full, i, 108);
      if (!ok) break;
      TF_AFTER();
      tf_add(tmem_o + lanes + (unsigned)(half * 32), keep, sum);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    if (ok) {  // the weights' sum over both halves
      float *both = stat + (tiles & 1) * 256 + r;
      both[half * 128] = l;
      __syncwarp();
      if (lane == 0) mbar_arrive(halves(q));
      ok = TF_WAIT(halves(q), tiles, 110);
      l = both[0] + both[128];
    }
    ok = __all_sync(0xffffffffu, ok && !*abort_flag);
    const bool empty = row_end <= row_lo;
    if (row < a.n) {
      tf_store_sums(a.o1, at.stream * a.o1.s + (long long)row * a.o1.r + at.head * a.o1.h, a, oh * 64 + half * 32, sum,
                    !ok ? NAN : empty ? 0.f : 1.0f / l);
      if (half == 0 && oh == 0)
        a.lse[((long long)at.stream * a.heads + at.head) * a.n + row] =
            !ok ? NAN : empty ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
    }
  }
  __syncwarp();
  pdl_launch_dependents();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    TF_AFTER();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_s), "r"(256u));
  }
}

// ---- dk and dv ------------------------------------------------------------------------------------------------------------------

template <int H>
__device__ __forceinline__ void tf_dkv(const CUtensorMap &map_q, const CUtensorMap &map_k, const CUtensorMap &map_v,
                                       const CUtensorMap &map_do, const TtArgs &a, int block) {
  extern __shared__ unsigned char smem_raw[];
  const unsigned base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char *base_ptr = smem_raw + (base - smem_u32(smem_raw));
  const unsigned k_off = base, v_off = base + TF_TILE, q_off = base + 2 * TF_TILE, do_off = base + 3 * TF_TILE, bars = base + TF_BAR_OFF;
  float *stat = reinterpret_cast<float *>(base_ptr + TF_STAT_OFF);  // [2][lse, delta][128]
  const unsigned kv_full = bars + 64, q_full = bars + 72, do_full = bars + 80, stat_full = bars + 88, s_full = bars + 96, p_ready = bars + 104,
                 dp_full = bars + 112, ds_ready = bars + 120, dv_full = bars + 128, dk_full = bars + 136;
  volatile unsigned *tmem_holder = reinterpret_cast<volatile unsigned *>(base_ptr + TF_BAR_OFF + 240);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(base_ptr + TF_BAR_OFF + 244);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int oh = H == 2 ? block & 1 : 0;  // which 64 dimensions of the result
  const TtPlace at = tt_place(a, a.groups, false, H, block);
  const int j0 = at.tile * TT_B, j1 = min(j0 + TT_B, at.keys);
  // rows that see a key of this tile: from lo on, to row_end
  const int lo = a.span.causal ? max(0, j0 - a.span.first) / TT_B * TT_B : 0;
  const long long past = a.span.window > 0 ? (long long)j1 - 1 + a.span.window - a.span.first : a.n;
  const int row_end = past < a.n ? (int)max(past, 0LL) : a.n;
  const int each = j0 < at.keys && row_end > lo ? (row_end - lo + TT_B - 1) / TT_B : 0;  // tiles per query head
  const int tiles = each * a.share;

  if (threadIdx.x == 0) {
    for (unsigned bar : {kv_full, q_full, do_full, stat_full, s_full, dp_full, dv_full, dk_full}) mbar_init(bar, 1);
    mbar_init(p_ready, 8);
    mbar_init(ds_ready, 8);
    if (H == 2)
      for (int i = 0; i < 8; ++i) mbar_init(bars + 8u * i, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) tt_alloc(tmem_holder, 512u);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  TF_AFTER();
  const unsigned tmem_s = *tmem_holder, tmem_dp = tmem_s + 192, tmem_dv = tmem_s + 384, tmem_dk = tmem_s + 448;
  pdl_wait();

  if (warp == 0) {
    TfRing ring{base, bars};
    int it = 0;
    bool ok = true;
    if (H == 1 && lane == 0 && tiles > 0) {
      mbar_expect_tx(kv_full, 2u * TF_TILE);
      tf_load(k_off, &map_k, j0, at.stream * a.groups + at.head, a.streams * a.groups, kv_full);
      tf_load(v_off, &map_v, j0, at.stream * a.groups + at.head, a.streams * a.groups, kv_full);
    }
    for (int h = at.head * a.share; h < (at.head + 1) * a.share && ok; ++h) {
      const int query_head = at.stream * a.heads + h;
      const long long stats = (long long)query_head * a.n;
      for (int t = 0; t < each; ++t, ++it) {
        const int r0 = lo + t * TT_B, st = it & 1;
        // (the statistics' other buffer may be read while this one is filled: the tile before last is done)
        if (it > 0) ok = TF_WAIT(dk_full, it - 1, 111);
        if (!ok) break;
        if (H == 1 && lane == 0) {
          mbar_expect_tx(q_full, TF_TILE);
          tf_load(q_off, &map_q, r0, query_head, a.streams * a.heads, q_full);
          mbar_expect_tx(do_full, TF_TILE);
          tf_load(do_off, &map_do, r0, query_head, a.streams * a.heads, do_full);
        }
        // a row that does not exist or sees no key has no weights: 2^(s - infinity)
#pragma unroll
        for (int e = lane; e < TT_B; e += 32) {
          const int row = r0 + e;
          const float z = row < a.n ? a.lse[stats + row] : -INFINITY;
          stat[st * 256 + e] = z == -INFINITY ? INFINITY : z * TT_LOG2E;
          stat[st * 256 + 128 + e] = row < a.n ? a.delta[stats + row] : 0.f;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(stat_full);
        __syncwarp();
        if constexpr (H == 2) {
          const int key_head = at.stream * a.groups + at.head, queries = a.streams * a.heads, keys = a.streams * a.groups;
          for (int d = 0; d < 2 && ok; ++d)
            ok = tf_put(ring, &map_k, d * 64, j0, key_head, keys, lane, abort_flag) &&
                 tf_put(ring, &map_q, d * 64, r0, query_head, queries, lane, abort_flag);
          for (int d = 0; d < 2 && ok; ++d)
            ok = tf_put(ring, &map_v, d * 64, j0, key_head, keys, lane, abort_flag) &&
                 tf_put(ring, &map_do, d * 64, r0, query_head, queries, lane, abort_flag);
          ok = ok && tf_put(ring, &map_do, oh * 64, r0, query_head, queries, lane, abort_flag) &&
               tf_put(ring, &map_q, oh * 64, r0, query_head, queries, lane, abort_flag);
          if (!ok) break;
        }
      }
    }
    if (H == 2) {
      if (*abort_flag) tf_drain(ring);
    } else if (*abort_flag && tiles > 0) {  // copies in flight must land before the shared memory goes away
      const unsigned long long limit = global_timer() + WAIT_LIMIT_NS;
      while (!mbar_try_wait(kv_full, 0) && global_timer() < limit) {}
      while (it > 0 && !mbar_try_wait(q_full, (unsigned)(it - 1) & 1u) && global_timer() < limit) {}
      while (it > 0 && !mbar_try_wait(do_full, (unsigned)(it - 1) & 1u) && global_timer() < limit) {}
    }
  } else if (warp == 1) {
    const int cols = H == 2 ? 64 : (a.dim + 15) & ~15;
    const unsigned idesc_s = umma_idesc_bf16(TT_B), idesc_d = umma_idesc_bf16(cols) | UMMA_B_MN_MAJOR;
    bool ok = H == 2 || tiles == 0 ? true : TF_WAIT(kv_full, 0, 112);
    int i = 0;
    TfRing ring{base, bars};
    for (; i < tiles && ok; ++i) {
      if constexpr (H == 2) {
        ok = tf_mma_ring(ring, tmem_s, idesc_s, s_full, abort_flag) && tf_mma_ring(ring, tmem_dp, idesc_s, dp_full, abort_flag) &&
             TF_WAIT(p_ready, i, 115) && tf_mma_ring_weights(ring, tmem_dv, tmem_s, idesc_d, dv_full, abort_flag) &&
             TF_WAIT(ds_ready, i, 116) && tf_mma_ring_weights(ring, tmem_dk, tmem_dp, idesc_d, dk_full, abort_flag);
        continue;
      }
      ok = TF_WAIT(q_full, i, 113);
      if (!ok) break;
      TF_AFTER();
      if (tc_elect()) {
        tf_mma_rows(tmem_s, k_off, q_off, idesc_s);
        tc_commit(s_full);
      }
      __syncwarp();
      ok = TF_WAIT(do_full, i, 114);
      if (!ok) break;
      if (tc_elect()) {
        tf_mma_rows(tmem_dp, v_off, do_off, idesc_s);
        tc_commit(dp_full);
      }
      __syncwarp();
      ok = TF_WAIT(p_ready, i, 115);
      if (!ok) break;
      TF_AFTER();
      if (tc_elect()) {
        tf_mma_weights(tmem_dv, tmem_s, do_off, idesc_d);
        tc_commit(dv_full);
      }
      __syncwarp();
      ok = TF_WAIT(ds_ready, i, 116);
      if (!ok) break;
      TF_AFTER();
      if (tc_elect()) {
        tf_mma_weights(tmem_dk, tmem_dp, q_off, idesc_d);
        tc_commit(dk_full);
      }
      __syncwarp();
    }
    if (!ok) {  // a bounded chance for the tensor pipe to finish before tensor memory is freed
      if (tc_elect()) tc_commit(dk_full);
      __syncwarp();
      const unsigned long long limit = global_timer() + WAIT_LIMIT_NS;
      while (!mbar_try_wait(dk_full, (unsigned)i & 1u) && global_timer() < limit) {}
    }
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    const unsigned lanes = (unsigned)(q * 32) << 16;
    const int key = j0 + q * 32 + lane;
    const bool key_live = key < at.keys;
    float dk[32], dv[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) dk[j] = dv[j] = 0.f;
    bool ok = true;
    for (int i = 0; i < tiles && ok; ++i) {
      const int st = i & 1, r0 = lo + i % each * TT_B + half * 64;
      // rows r0 + c that see this key: [c_lo, c_end)
      const int c_lo = a.span.causal ? key - a.span.first - r0 : 0;
      const long long pe = a.span.window > 0 ? (long long)key + a.span.window - a.span.first - r0 : 64;
      const int c_end = !key_live ? 0 : pe < 64 ? (int)max(pe, 0LL) : 64;
      const bool inside = __all_sync(0xffffffffu, c_lo <= 0 && c_end >= 64);
      ok = TF_WAIT(stat_full, i, 117) && TF_WAIT(s_full, i, 118);
      if (!ok) break;
      TF_AFTER();
      float p[64];
      {
        unsigned(&u)[2][32] = reinterpret_cast<unsigned(&)[2][32]>(p);
        tc_ld32(tmem_s + lanes + (unsigned)(half * 64), u[0]);
        tc_ld32(tmem_s + lanes + (unsigned)(half * 64 + 32), u[1]);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      }
      const float4 *z = reinterpret_cast<const float4 *>(stat + st * 256 + half * 64);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float4 v = z[j];
        p[4 * j] = tt_exp2(fmaf(p[4 * j], a.factor, -v.x));
        p[4 * j + 1] = tt_exp2(fmaf(p[4 * j + 1], a.factor, -v.y));
        p[4 * j + 2] = tt_exp2(fmaf(p[4 * j + 2], a.factor, -v.z));
        p[4 * j + 3] = tt_exp2(fmaf(p[4 * j + 3], a.factor, -v.w));
      }
      if (!inside) {
#pragma unroll
        for (int j = 0; j < 64; ++j)
          if (j < c_lo || j >= c_end) p[j] = 0.f;
      }
      tf_store_parts(tmem_s + lanes, half, 0, p);
      tf_store_parts(tmem_s + lanes, half, 32, p + 32);
      TF_READY(p_ready);
      ok = TF_WAIT(dp_full, i, 119);
      if (!ok) break;
      TF_AFTER();
      const float4 *de = reinterpret_cast<const float4 *>(stat + st * 256 + 128 + half * 64);
      {  // all of the half's columns first: the parts lie over them
        unsigned u[2][32];
        tc_ld32(tmem_dp + lanes + (unsigned)(half * 64), u[0]);
        tc_ld32(tmem_dp + lanes + (unsigned)(half * 64 + 32), u[1]);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 v = de[(c * 32 + j) >> 2];
            p[c * 32 + j] *= __uint_as_float(u[c][j]) - v.x;
            p[c * 32 + j + 1] *= __uint_as_float(u[c][j + 1]) - v.y;
            p[c * 32 + j + 2] *= __uint_as_float(u[c][j + 2]) - v.z;
            p[c * 32 + j + 3] *= __uint_as_float(u[c][j + 3]) - v.w;
          }
        if (!inside) {  // (a weight of zero has no part even where the other factor is not finite)
#pragma unroll
          for (int j = 0; j < 64; ++j)
            if (j < c_lo || j >= c_end) p[j] = 0.f;
        }
      }
      tf_store_parts(tmem_dp + lanes, half, 0, p);
      tf_store_parts(tmem_dp + lanes, half, 32, p + 32);
      TF_READY(ds_ready);
      ok = TF_WAIT(dv_full, i, 120);
      if (!ok) break;
      TF_AFTER();
      tf_add(tmem_dv + lanes + (unsigned)(half * 32), 1.f, dv);
      ok = TF_WAIT(dk_full, i, 121);
      if (!ok) break;
      TF_AFTER();
      tf_add(tmem_dk + lanes + (unsigned)(half * 32), 1.f, dk);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    ok = __all_sync(0xffffffffu, ok && !*abort_flag);
    if (key < a.m) {
      tf_store_sums(a.o1, at.stream * a.o1.s + (long long)key * a.o1.r + at.head * a.o1.h, a, oh * 64 + half * 32, dk, ok ? a.scale : NAN);
      tf_store_sums(a.o2, at.stream * a.o2.s + (long long)key * a.o2.r + at.head * a.o2.h, a, oh * 64 + half * 32, dv, ok ? 1.f : NAN);
    }
  }
  __syncwarp();
  pdl_launch_dependents();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    TF_AFTER();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_s), "r"(512u));
  }
}

// ---- dq -------------------------------------------------------------------------------------------------------------------------

template <int H>
__device__ __forceinline__ void tf_dq(const CUtensorMap &map_q, const CUtensorMap &map_k, const CUtensorMap &map_v,
                                      const CUtensorMap &map_do, const TtArgs &a, int block) {
  extern __shared__ unsigned char smem_raw[];
  const unsigned base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char *base_ptr = smem_raw + (base - smem_u32(smem_raw));
  const unsigned q_off = base, do_off = base + TF_TILE, k_off = base + 2 * TF_TILE, v_off = base + 3 * TF_TILE, bars = base + TF_BAR_OFF;
  const unsigned q_full = bars + 64, k_full = bars + 72, v_full = bars + 80, s_full = bars + 88, dp_full = bars + 96, ds_ready = bars + 104,
                 dq_full = bars + 112;
  volatile unsigned *tmem_holder = reinterpret_cast<volatile unsigned *>(base_ptr + TF_BAR_OFF + 240);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(base_ptr + TF_BAR_OFF + 244);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int oh = H == 2 ? block & 1 : 0;  // which 64 dimensions of the result
  const TtPlace at = tt_place(a, a.heads, a.span.causal != 0, H, block);
  const int r0 = at.tile * TT_B, r1 = min(r0 + TT_B, a.n), kh = at.head / a.share;
  const int lo = a.span.lo(r0), end = a.span.end(r1 - 1, at.keys);
  const int tiles = end > lo ? (end - lo + TT_B - 1) / TT_B : 0;

  if (threadIdx.x == 0) {
    for (unsigned bar : {q_full, k_full, v_full, s_full, dp_full, dq_full}) mbar_init(bar, 1);
    mbar_init(ds_ready, 8);
    if (H == 2)
      for (int i = 0; i < 8; ++i) mbar_init(bars + 8u * i, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) tt_alloc(tmem_holder, 512u);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  TF_AFTER();
  const unsigned tmem_s = *tmem_holder, tmem_dp = tmem_s + 128, tmem_dq = tmem_s + 320;
  pdl_wait();

  if (warp == 0) {
    if constexpr (H == 2) {
      TfRing ring{base, bars};
      const int query_head = at.stream * a.heads + at.head, key_head = at.stream * a.groups + kh;
      const int queries = a.streams * a.heads, keys = a.streams * a.groups;
      bool ok = true;
      for (int i = 0; i < tiles && ok; ++i) {
        const int j0 = lo + i * TT_B;
        for (int d = 0; d < 2 && ok; ++d)
          ok = tf_put(ring, &map_do, d * 64, r0, query_head, queries, lane, abort_flag) &&
               tf_put(ring, &map_v, d * 64, j0, key_head, keys, lane, abort_flag);
        for (int d = 0; d < 2 && ok; ++d)
          ok = tf_put(ring, &map_q, d * 64, r0, query_head, queries, lane, abort_flag) &&
               tf_put(ring, &map_k, d * 64, j0, key_head, keys, lane, abort_flag);
        ok = ok && tf_put(ring, &map_k, oh * 64, j0, key_head, keys, lane, abort_flag);
      }
      if (*abort_flag) tf_drain(ring);
    } else {
    int it = 0;
    bool ok = true;
    const int query_head = at.stream * a.heads + at.head, key_head = at.stream * a.groups + kh;
    if (lane == 0 && tiles > 0) {
      mbar_expect_tx(q_full, 2u * TF_TILE);
      tf_load(q_off, &map_q, r0, query_head, a.streams * a.heads, q_full);
      tf_load(do_off, &map_do, r0, query_head, a.streams * a.heads, q_full);
    }
    for (; it < tiles; ++it) {
      const int j0 = lo + it * TT_B;
      if (it > 0) ok = TF_WAIT(dp_full, it - 1, 131);  // dout v has read the values
      if (!ok) break;
      if (lane == 0) {
        mbar_expect_tx(v_full, TF_TILE);
        tf_load(v_off, &map_v, j0, key_head, a.streams * a.groups, v_full);
      }
      __syncwarp();
      if (it > 0) ok = TF_WAIT(dq_full, it - 1, 132);  // dS k has read the keys
      if (!ok) {
        ++it;  // (its values are on their way)
        break;
      }
      if (lane == 0) {
        mbar_expect_tx(k_full, TF_TILE);
        tf_load(k_off, &map_k, j0, key_head, a.streams * a.groups, k_full);
      }
      __syncwarp();
    }
    if (*abort_flag && tiles > 0) {  // copies in flight must land before the shared memory goes away
      const unsigned long long limit = global_timer() + WAIT_LIMIT_NS;
      while (!mbar_try_wait(q_full, 0) && global_timer() < limit) {}
      while (it > 0 && !mbar_try_wait(v_full, (unsigned)(it - 1) & 1u) && global_timer() < limit) {}
      const int k_loads = ok ? it : it - 1;
      while (k_loads > 0 && !mbar_try_wait(k_full, (unsigned)(k_loads - 1) & 1u) && global_timer() < limit) {}
    }
    }
  } else if (warp == 1) {
    const int cols = H == 2 ? 64 : (a.dim + 15) & ~15;
    const unsigned idesc_s = umma_idesc_bf16(TT_B), idesc_d = umma_idesc_bf16(cols) | UMMA_B_MN_MAJOR;
    bool ok = H == 2 || tiles == 0 ? true : TF_WAIT(q_full, 0, 133);
    int i = 0;
    TfRing ring{base, bars};
    for (; i < tiles && ok; ++i) {
      if constexpr (H == 2) {
        ok = tf_mma_ring(ring, tmem_dp, idesc_s, dp_full, abort_flag) && tf_mma_ring(ring, tmem_s, idesc_s, s_full, abort_flag) &&
             TF_WAIT(ds_ready, i, 136) && tf_mma_ring_weights(ring, tmem_dq, tmem_dp, idesc_d, dq_full, abort_flag);
        continue;
      }
      ok = TF_WAIT(v_full, i, 134);
      if (!ok) break;
      TF_AFTER();
      // (over dP and its parts: dS k of the tile before has read them, in the order of issue; over S: read before ds_ready)
      if (tc_elect()) {
        tf_mma_rows(tmem_dp, do_off, v_off, idesc_s);
        tc_commit(dp_full);
      }
      __syncwarp();
      ok = TF_WAIT(k_full, i, 135);
      if (!ok) break;
      if (tc_elect()) {
        tf_mma_rows(tmem_s, q_off, k_off, idesc_s);
        tc_commit(s_full);
      }
      __syncwarp();
      ok = TF_WAIT(ds_ready, i, 136);
      if (!ok) break;
      TF_AFTER();
      if (tc_elect()) {
        tf_mma_weights(tmem_dq, tmem_dp, k_off, idesc_d);
        tc_commit(dq_full);
      }
      __syncwarp();
    }
    if (!ok) {  // a bounded chance for the tensor pipe to finish before tensor memory is freed
      if (tc_elect()) tc_commit(dq_full);
      __syncwarp();
      const unsigned long long limit = global_timer() + WAIT_LIMIT_NS;
      while (!mbar_try_wait(dq_full, (unsigned)i & 1u) && global_timer() < limit) {}
    }
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    const unsigned lanes = (unsigned)(q * 32) << 16;
    const int row = r0 + q * 32 + lane;
    const int row_lo = a.span.lo(row), row_end = a.span.end(row, at.keys);
    const int warp_lo = a.span.lo(r0 + q * 32 + 31), warp_end = a.span.end(r0 + q * 32, at.keys);
    const long long x = ((long long)at.stream * a.heads + at.head) * a.n + row;
    const float z = row < a.n ? a.lse[x] : -INFINITY, delta = row < a.n ? a.delta[x] : 0.f;
    const float lse = z == -INFINITY ? INFINITY : z * TT_LOG2E;  // a row that sees no key has no weights: 2^(s - infinity)
    float sum[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) sum[j] = 0.f;
    bool ok = true;
    for (int i = 0; i < tiles && ok; ++i) {
      const int j0 = lo + i * TT_B + half * 64;
      const int c_lo = row_lo - j0, c_end = row_end - j0;
      const bool inside = warp_lo <= j0 && warp_end >= j0 + 64;
      ok = TF_WAIT(s_full, i, 137) && TF_WAIT(dp_full, i, 138);
      if (!ok) break;
      TF_AFTER();
      float p[64];
      {
        unsigned(&v)[2][32] = reinterpret_cast<unsigned(&)[2][32]>(p);
        tc_ld32(tmem_s + lanes + (unsigned)(half * 64), v[0]);
        tc_ld32(tmem_s + lanes + (unsigned)(half * 64 + 32), v[1]);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      }
#pragma unroll
      for (int c = 0; c < 64; c += 32) {  // all of the half's columns before the parts go over them
        unsigned u[32];
        tc_ld32(tmem_dp + lanes + (unsigned)(half * 64 + c), u);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int j = 0; j < 32; ++j) p[c + j] = tt_exp2(fmaf(p[c + j], a.factor, -lse)) * (__uint_as_float(u[j]) - delta);
      }
      if (!inside) {
#pragma unroll
        for (int j = 0; j < 64; ++j)
          if (j < c_lo || j >= c_end) p[j] = 0.f;
      }
      tf_store_parts(tmem_dp + lanes, half, 0, p);
      tf_store_parts(tmem_dp + lanes, half, 32, p + 32);
      TF_READY(ds_ready);
      ok = TF_WAIT(dq_full, i, 139);
      if (!ok) break;
      TF_AFTER();
      tf_add(tmem_dq + lanes + (unsigned)(half * 32), 1.f, sum);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    ok = __all_sync(0xffffffffu, ok && !*abort_flag);
    if (row < a.n)
      tf_store_sums(a.o1, at.stream * a.o1.s + (long long)row * a.o1.r + at.head * a.o1.h, a, oh * 64 + half * 32, sum, ok ? a.scale : NAN);
  }
  __syncwarp();
  pdl_launch_dependents();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    TF_AFTER();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_s), "r"(512u));
  }
}

// Both, in one launch: neither waits for the other, and few rows leave multiprocessors free (4 streams of 64 rows: 14 and 16 us one behind
// the other).
template <int H>
__global__ void __launch_bounds__(TF_THREADS, 1)
train_backward_f32_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                          const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do,
                          const __grid_constant__ TtArgs by_keys, const __grid_constant__ TtArgs by_rows, int blocks) {
  const int block = (int)blockIdx.x;
  if (block < blocks) tf_dkv<H>(map_q, map_k, map_v, map_do, by_keys, block);
  else tf_dq<H>(map_q, map_k, map_v, map_do, by_rows, block - blocks);
}

// ---- host -----------------------------------------------------------------------------------------------------------------------

size_t part_bytes(long long streams, long long heads, long long rows, long long dim) {
  return (size_t)(streams * heads * rows) * (dim > 64 ? 128 : 64) * 3 * 2;
}

bool rows16(const HeadView &x) {
  return x.c == 1 && reinterpret_cast<uintptr_t>(x.p) % 16 == 0 && x.s % 4 == 0 && x.r % 4 == 0 && x.h % 4 == 0;
}

struct Parts {
  bf16 *p;
  int streams, rows, heads, dim;
};

CUtensorMap part_map(const Parts &x) {
  CUtensorMap map;
  const unsigned long long cols = x.dim > 64 ? 128 : 64;
  const unsigned long long extent[4] = {cols, 1, (unsigned long long)x.rows, 3ull * x.streams * x.heads};
  const unsigned long long strides[3] = {cols * 2, cols * 2, (unsigned long long)x.rows * cols * 2};
  tc_make_map_heads(&map, x.p, extent, strides, TT_B);
  return map;
}

// The operands' parts into the workspace, delta too where it is wanted.
void split(const TrainAttention &a, char *work, float *delta, Parts (&parts)[4], cudaStream_t st) {
  TfSplit g{};
  g.count = delta ? 4 : 3;
  g.streams = a.streams;
  g.dim = a.dim;
  g.chunks = a.dim > 64 ? 16 : 8;
  g.seen = a.seen;
  g.span = TrainSpan{a.first, a.window, a.causal};
  g.lengths = a.lengths;
  g.out = a.out;
  g.delta = delta;
  long long blocks = 0;
  const HeadView *views[4] = {&a.q, &a.k, &a.v, &a.dout};
  for (int i = 0; i < g.count; ++i) {
    const bool keys = i == 1 || i == 2;
    TfTensor &t = g.t[i];
    t.x = *views[i];
    t.rows = keys ? a.m : a.n;
    t.heads = keys ? a.groups : a.heads;
    t.keys = keys;
    t.vec = rows16(t.x);
    t.part = reinterpret_cast<bf16 *>(work);
    const int each = 256 / g.chunks;
    const long long b = (long long)a.streams * t.heads * ((t.rows + each - 1) / each);
    blocks += b;
    if (blocks > 0x7fffffffLL || 3LL * a.streams * t.heads > 0x7fffffffLL)
      throw std::invalid_argument("attention: too many rows, heads and streams for one call");
    t.blocks = (int)b;
    parts[i] = Parts{t.part, a.streams, t.rows, t.heads, a.dim};
    work += part_bytes(a.streams, t.heads, t.rows, a.dim);
  }
  train_split_kernel<<<(unsigned)blocks, 256, 0, st>>>(g);
  LB_LAUNCH_CHECK();
}

}  // namespace

size_t train_attention_f32_workspace(long long streams, long long n, long long m, long long heads, long long groups, long long dim,
                                     bool backward) {
  return (backward ? 2 : 1) * part_bytes(streams, heads, n, dim) + 2 * part_bytes(streams, groups, m, dim);
}

namespace {

template <int H>
void forward(const TrainAttention &a, const Parts (&p)[4], cudaStream_t st) {
  TtArgs t = tt_args(a, a.n);
  t.o1 = a.out;
  t.vec = rows16(a.out);
  static SharedMemoryOnce once;
  once.set(train_forward_f32_kernel<H>, TF_SMEM);
  launch_pdl(train_forward_f32_kernel<H>, dim3(tt_grid(t, a.heads, H)), dim3(TF_THREADS), TF_SMEM, st, true, part_map(p[0]),
             part_map(p[1]), part_map(p[2]), t);
}

template <int H>
void backward(const TrainAttention &a, float *delta, const Parts (&p)[4], cudaStream_t st) {
  const CUtensorMap mq = part_map(p[0]), mk = part_map(p[1]), mv = part_map(p[2]), md = part_map(p[3]);
  TtArgs t = tt_args(a, a.m);
  t.delta = delta;
  t.o1 = a.dk;
  t.o2 = a.dv;
  t.vec = rows16(a.dk) && rows16(a.dv);
  TtArgs u = tt_args(a, a.n);
  u.delta = delta;
  u.o1 = a.dq;
  u.vec = rows16(a.dq);
  const unsigned by_keys = tt_grid(t, a.groups, H), by_rows = tt_grid(u, a.heads, H);
  if (by_rows > 0x7fffffffu - by_keys) throw std::invalid_argument("attention: too many rows, heads and streams for one call");
  static SharedMemoryOnce once;
  once.set(train_backward_f32_kernel<H>, TF_SMEM);
  launch_pdl(train_backward_f32_kernel<H>, dim3(by_keys + by_rows), dim3(TF_THREADS), TF_SMEM, st, true, mq, mk, mv, md, t, u,
             (int)by_keys);
}

}  // namespace

void launch_train_attention_forward_f32(const TrainAttention &a, void *work, cudaStream_t st) {
  Parts p[4];
  split(a, static_cast<char *>(work), nullptr, p, st);
  if (a.dim <= 64) forward<1>(a, p, st);
  else forward<2>(a, p, st);
}

void launch_train_attention_backward_f32(const TrainAttention &a, float *delta, void *work, cudaStream_t st) {
  Parts p[4];
  split(a, static_cast<char *>(work), delta, p, st);
  if (a.dim <= 64) backward<1>(a, delta, p, st);
  else backward<2>(a, delta, p, st);
}

}  // namespace lb

// Orthogonalised momentum: the update of a weight matrix by the polynomial iteration
//   X = U / (|U| + 1e-7),  X <- a X + (b A + c A^2) X,  A = X X^T,  (a, b, c) = (3.4445, -4.7750, 2.0315)
// in the space of the matrix's smaller side (X <- X (b A + c A^2) + a X with A = X^T X for a tall one), which drives its singular
// values towards 1 (a Newton-Schulz iteration; the quintic's coefficients as K. Jordan published them with this optimiser in 2024);
// and the optimiser step with it,
//   momentum <- mu momentum + grad,  U = grad + mu momentum or momentum,
//   params <- (1 - lr decay) params - lr sqrt(max(1, m / n)) X.
// All matrices of a call have one shape and go through each product together.
//
// A step is three products: A = X X^T, B = b A + c A A, X <- a X + B X. The matrix that is added is the first term of the sum that a
// thread keeps in registers, so nothing of it is lost to the tensor pipe's truncation (with a on B's diagonal instead the result
// of two steps was 13 times as far from 64 bits as by 32-bit products; so 2).
//
// Matrices live as pairs of fp16 values: z 2^e = hi + 2^-11 lo, 22 bits, with one exponent e per matrix, kind and step. It follows
// from a bound on the singular values alone: those of X_k are at most min(1.25, rho a^k) where rho = |X_0| (the polynomial stays
// below 1.21 on [0, 1.21] and below a s), those of A at most its square, of B min(2.85, |b| of that). No entry is larger, and e puts
// the bound at 2^13 to 2^14. A product is three: hi lo and lo hi, then, scaled by 2^-11 in the instruction that starts it, hi hi on top; lo lo is below
// 2^-22 of a term, mostly far below, and left out. The tensor pipe truncates when it adds, so chains in tensor memory are 64 k long and are added in
// registers, rounded to nearest.
//
// One persistent kernel for the three products of a step, tiles of 128 x 128: warp 0 issues TMA (stages of 64 k: four tiles of 16
// KB), warp 1 owns tensor memory and issues the MMAs, eight warps add finished chains (a thread: a row and half of the columns) and
// store through patches of shared memory that TMA carries out (a pair's threads, with 128 columns, spill 116 to 176 bytes). Nothing is transposed in memory: an operand whose rows run along k
// is read as it lies (M or N contiguous). A and B are symmetric: tiles up to the diagonal are multiplied, and stored on both
// sides of it.
// Every wait is bounded; one that runs out ends the CTA, whose results are then NaN. Pairs of CTAs share a tile of 256 rows where there are tiles for all SMs, clusters of up
// to eight a tile's range of k where there are few; no multicast.
#include "train_ops.cuh"
#include "gemm_tc.cuh"
#include "tc_ptx.cuh"

#include <cuda_fp16.h>

namespace lb {

namespace {

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f, NS_EPS = 1e-7f;
constexpr double NS_SPLIT = 2.0;
constexpr int NS_PARTS = 256;  // partial sums of a matrix's norm, at most
constexpr int NS_THREADS = 320, NS_LD = 132;  // floats between rows of a finished range of k

struct Pair {
  __half *hi, *lo;  // [count][rows][ld]
};

struct NsWork {
  double *parts;   // [count][NS_PARTS]
  float *rho;      // [count]
  Pair x[2], a, b;
  long long ldx, ldp;
};

// Exponents of the pairs of X, A and B in step k.
__device__ __forceinline__ int ns_exponent(float bound) {
  if (!(bound > 0.f)) return 0;
  const int e = 13 - ilogbf(bound);
  return e < 100 ? e : 100;
}
__device__ __forceinline__ float ns_bound(float rho, int k) {
  for (int i = 0; i < k; ++i) rho *= 3.45f;
  return fminf(1.25f, rho);
}
__device__ __forceinline__ int ns_exp_x(float rho, int k) { return ns_exponent(ns_bound(rho, k)); }
__device__ __forceinline__ int ns_exp_a(float rho, int k) {
  const float s = ns_bound(rho, k);
  return ns_exponent(s * s);
}
__device__ __forceinline__ int ns_exp_b(float rho, int k) {
  const float s = ns_bound(rho, k);
  return ns_exponent(fminf(2.85f, 4.8f * s * s));
}

// Two values, already scaled, as pairs: a conversion of two costs what one does.
__device__ __forceinline__ void ns_split2(float a, float b, unsigned &hi, unsigned &lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn((a - f.x) * 2048.f, (b - f.y) * 2048.f);
  hi = *reinterpret_cast<const unsigned *>(&h);
  lo = *reinterpret_cast<const unsigned *>(&l);
}
__device__ __forceinline__ float ns_value(__half hi, __half lo) { return fmaf(__half2float(lo), 1.f / 2048.f, __half2float(hi)); }
__device__ __forceinline__ float ns_pow2(int e) { return ldexpf(1.f, e); }

// ---- momentum and norm, first pair, end ------------------------------------------------------------------------------------------

__device__ __forceinline__ float *element(const MatView &v, long long batch_off, long long r, long long c) {
  return reinterpret_cast<float *>(v.data + batch_off + r * v.rs + c * v.cs);
}

// Four elements of a row from column c on; `vec`: rows of the view on 16-byte boundaries. What lies behind the row is 0.
// FLAT: a matrix whose rows follow one another, as one row.
template <bool FLAT>
__device__ __forceinline__ void load4(const MatView &v, long long off, long long r, long long c, bool vec, float (&x)[4]) {
  const float *p = FLAT ? reinterpret_cast<float *>(v.data + off) + c : element(v, off, r, c);
  if (FLAT || (vec && c + 4 <= v.cols)) {
    const float4 f = *reinterpret_cast<const float4 *>(p);
    x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = c + j < v.cols ? *reinterpret_cast<const float *>(reinterpret_cast<const char *>(p) + j * v.cs) : 0.f;
  }
}
template <bool FLAT>
__device__ __forceinline__ void store4(const MatView &v, long long off, long long r, long long c, bool vec, const float (&x)[4]) {
  float *p = FLAT ? reinterpret_cast<float *>(v.data + off) + c : element(v, off, r, c);
  if (FLAT || (vec && c + 4 <= v.cols)) {
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < v.cols) *reinterpret_cast<float *>(reinterpret_cast<char *>(p) + j * v.cs) = x[j];
  }
}

__device__ __forceinline__ double ns_block_sum(double s) {
  __shared__ double red[8];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = red[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) s += red[i];
  return s;
}

enum { VEC_G = 1, VEC_M = 2, VEC_P = 4 };

// Four groups of four elements at a time and thread, so that their loads are in flight together (with one a step on six matrices of
// 512 x 2048 took 383 us, with four 375).
constexpr int NS_AHEAD = 4;
template <bool FLAT, typename F>
__device__ __forceinline__ void for_quads(long long rows, long long quads, F f) {
  const long long all = rows * quads, step = 256LL * gridDim.x;
  for (long long e0 = blockIdx.x * 256LL + threadIdx.x; e0 < all; e0 += NS_AHEAD * step) {
    long long r[NS_AHEAD], c[NS_AHEAD];
    int n = 0;
#pragma unroll
    for (int i = 0; i < NS_AHEAD; ++i) {
      const long long e = e0 + i * step < all ? e0 + i * step : e0;  // (a group past the end is the first one's again, and not used)
      r[i] = FLAT ? 0 : div_index(e, quads);
      c[i] = (e - r[i] * quads) * 4;
      n += e0 + i * step < all;
    }
    f(r, c, n);
  }
}

template <bool FLAT>
__global__ void __launch_bounds__(256) muon_begin_kernel(const __grid_constant__ MuonStep g, NsWork w, unsigned vec) {
  pdl_launch_dependents();
  pdl_wait();
  const long long batch = blockIdx.y;
  const long long go = batch_offset(g.grads, batch), mo = g.step ? batch_offset(g.momentum, batch) : 0;
  double sum = 0.0;
  for_quads<FLAT>(g.grads.rows, (g.grads.cols + 3) / 4, [&](const long long(&r)[NS_AHEAD], const long long(&c)[NS_AHEAD], int n) {
    float u[NS_AHEAD][4], m[NS_AHEAD][4];
#pragma unroll
    for (int i = 0; i < NS_AHEAD; ++i) {
      load4<FLAT>(g.grads, go, r[i], c[i], vec & VEC_G, u[i]);
      if (g.step) load4<FLAT>(g.momentum, mo, r[i], c[i], vec & VEC_M, m[i]);
    }
#pragma unroll
    for (int i = 0; i < NS_AHEAD; ++i) {
      if (i >= n) break;
      if (g.step) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          m[i][j] = fmaf(g.mu, m[i][j], u[i][j]);
          u[i][j] = g.nesterov ? fmaf(g.mu, m[i][j], u[i][j]) : m[i][j];
        }
        store4<FLAT>(g.momentum, mo, r[i], c[i], vec & VEC_M, m[i]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += (double)u[i][j] * (double)u[i][j];
    }
  });
  sum = ns_block_sum(sum);
  if (threadIdx.x == 0) w.parts[batch * NS_PARTS + blockIdx.x] = sum;
}

template <bool FLAT>
__global__ void __launch_bounds__(256) muon_pair_kernel(const __grid_constant__ MuonStep g, NsWork w, unsigned vec, int parts) {
  pdl_launch_dependents();
  pdl_wait();
  const long long batch = blockIdx.y;
  const long long go = batch_offset(g.grads, batch), mo = g.step ? batch_offset(g.momentum, batch) : 0;
  const double norm = sqrt(ns_block_sum((int)threadIdx.x < parts ? w.parts[batch * NS_PARTS + threadIdx.x] : 0.0));
  const double inv = 1.0 / (norm + (double)NS_EPS);
  const float rho = (float)(norm * inv);
  if (blockIdx.x == 0 && threadIdx.x == 0) w.rho[batch] = rho;
  // x = u scale, by two factors: the second stays in the range of 32 bits whatever the norm
  const double scale = inv * (double)ns_pow2(ns_exp_x(rho, 0));
  const float first = scale < 1e-30 ? 5.421010862427522e-20f : 1.f, second = (float)(scale / (double)first);  // 2^-64
  __half *hi = w.x[0].hi + batch * g.grads.rows * w.ldx, *lo = w.x[0].lo + batch * g.grads.rows * w.ldx;
  for_quads<FLAT>(g.grads.rows, w.ldx / 4, [&](const long long(&r)[NS_AHEAD], const long long(&c)[NS_AHEAD], int n) {
    float u[NS_AHEAD][4], m[NS_AHEAD][4];
#pragma unroll
    for (int i = 0; i < NS_AHEAD; ++i) {
      const bool in = FLAT || c[i] < g.grads.cols;
#pragma unroll
      for (int j = 0; j < 4; ++j) u[i][j] = m[i][j] = 0.f;
      if (in) load4<FLAT>(g.grads, go, r[i], c[i], vec & VEC_G, u[i]);
      if (in && g.step) load4<FLAT>(g.momentum, mo, r[i], c[i], vec & VEC_M, m[i]);
    }
#pragma unroll
    for (int i = 0; i < NS_AHEAD; ++i) {
      if (i >= n) break;
      unsigned h[2], l[2];
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float v = !g.step ? u[i][j] : g.nesterov ? fmaf(g.mu, m[i][j], u[i][j]) : m[i][j];
        x[j] = v * first * second;
      }
      ns_split2(x[0], x[1], h[0], l[0]);
      ns_split2(x[2], x[3], h[1], l[1]);
      *reinterpret_cast<uint2 *>(hi + r[i] * w.ldx + c[i]) = make_uint2(h[0], h[1]);
      *reinterpret_cast<uint2 *>(lo + r[i] * w.ldx + c[i]) = make_uint2(l[0], l[1]);
    }
  });
}

template <bool FLAT>
__global__ void __launch_bounds__(256)
muon_end_kernel(const __grid_constant__ MuonStep g, NsWork w, unsigned vec, float keep, float rate) {
  pdl_launch_dependents();
  pdl_wait();
  const long long batch = blockIdx.y;
  const long long po = batch_offset(g.params, batch);
  const Pair x = w.x[g.steps & 1];
  const __half *hi = x.hi + batch * g.grads.rows * w.ldx, *lo = x.lo + batch * g.grads.rows * w.ldx;
  const float scale = ns_pow2(-ns_exp_x(w.rho[batch], g.steps));
  for_quads<FLAT>(g.grads.rows, (g.grads.cols + 3) / 4, [&](const long long(&r)[NS_AHEAD], const long long(&c)[NS_AHEAD], int n) {
    uint2 h[NS_AHEAD], l[NS_AHEAD];
    float p[NS_AHEAD][4];
#pragma unroll
    for (int i = 0; i < NS_AHEAD; ++i) {
      h[i] = *reinterpret_cast<const uint2 *>(hi + r[i] * w.ldx + c[i]);
      l[i] = *reinterpret_cast<const uint2 *>(lo + r[i] * w.ldx + c[i]);
      if (g.step) load4<FLAT>(g.params, po, r[i], c[i], vec & VEC_P, p[i]);
    }
#pragma unroll
    for (int i = 0; i < NS_AHEAD; ++i) {
      if (i >= n) break;
      const __half *hh = reinterpret_cast<const __half *>(&h[i]), *ll = reinterpret_cast<const __half *>(&l[i]);
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = ns_value(hh[j], ll[j]) * scale;
        if (g.step) v[j] = fmaf(-rate, v[j], p[i][j] * keep);
      }
      store4<FLAT>(g.params, po, r[i], c[i], vec & VEC_P, v);
    }
  });
}

// ---- the products of a step -------------------------------------------------------------------------------------------------------

// GRAM: A = X X^T or X^T X; POLY: B = b A + c A A; APPLY: X' = a X + B X or a X + X B
enum NsOp { GRAM, POLY, APPLY };

struct NsProduct {
  Pair add, out;         // A for POLY, X for APPLY; the result
  long long ld;          // of it and of the result
  int m, n, k;           // sizes of the product
  int m_tiles, n_tiles, tiles;  // tiles of all matrices
  int step;
  int splits;            // CTAs of a cluster that share a tile's range of k (SPLIT)
  const float *rho;
};

struct NsSmem {
  static constexpr int STAGES = 3, TILE = 16384, STAGE = 4 * TILE;
  static constexpr int PATCH_OFF = STAGES * STAGE, PATCH = 4096;  // 32 x 32 elements of hi and of lo, per storing warp
  static constexpr int BAR_OFF = PATCH_OFF + 8 * PATCH;
  static constexpr int TOTAL = BAR_OFF + 128 + 1024;
  static_assert(TOTAL <= 227 * 1024, "");
};

constexpr unsigned UMMA_A_MN_MAJOR = 1u << 15;

// Instructions of a pair of CTAs: the even one's thread issues them for both, operands at the same places of both shared memories
// (of the right operand each CTA holds half of the rows), rows 128 .. 255 of the result in the odd one's tensor memory.
template <bool PAIR>
__device__ __forceinline__ void ns_load(unsigned to, const CUtensorMap *map, int x, int z, int w, unsigned bar) {
  if constexpr (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(to), "l"(map), "r"(x), "r"(0), "r"(z), "r"(w), "r"(bar)
        : "memory");
  else tma_load_4d(to, map, x, 0, z, w, bar);
}
// D = A B, D += A B, or D = 2^-11 D + A B.
enum NsStart { NS_NEW, NS_ADD, NS_SCALED };
template <bool PAIR>
__device__ __forceinline__ void ns_mma(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, NsStart how) {
#define NS_MMA(group, scale)                                           \
  asm volatile("{\n\t.reg .pred p;\n\t"                                \
               "setp.ne.b32 p, %4, 0;\n\t"                             \
               "tcgen05.mma.cta_group::" group ".kind::f16 [%0], %1, %2, %3, p" scale ";\n\t}" \
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(how == NS_NEW ? 0u : 1u)              \
               : "memory")
  if (how == NS_SCALED) {
    if constexpr (PAIR) NS_MMA("2", ", 11");
    else NS_MMA("1", ", 11");
  } else {
    if constexpr (PAIR) NS_MMA("2", "");
    else NS_MMA("1", "");
  }
#undef NS_MMA
}
template <bool PAIR>
__device__ __forceinline__ void ns_commit(unsigned bar) {  // of a pair: the barrier at this place in both CTAs
  if constexpr (PAIR)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"((unsigned short)3)
                 : "memory");
  else tc_commit(bar);
}

template <NsOp OP, bool A_MN, bool B_MN, bool PAIR, bool SPLIT>
__global__ void __launch_bounds__(NS_THREADS, 1)
ns_product_kernel(const __grid_constant__ CUtensorMap map_ah, const __grid_constant__ CUtensorMap map_al,
                  const __grid_constant__ CUtensorMap map_bh, const __grid_constant__ CUtensorMap map_bl,
                  const __grid_constant__ CUtensorMap map_oh, const __grid_constant__ CUtensorMap map_ol,
                  const __grid_constant__ NsProduct g) {
  using L = NsSmem;
  constexpr int S = L::STAGES, CTAS = PAIR ? 2 : 1, T = 128 * CTAS;  // tiles of T x T by CTAS CTAs, 128 rows each
  constexpr int CHAINS = 4 / CTAS, COLS = 64 * CTAS;  // chains in flight, T columns of tensor memory each; columns of a thread
  constexpr bool SYM = OP != APPLY;
  static_assert(!(PAIR && SPLIT), "");
  const int rank = PAIR ? (int)blockIdx.x & 1 : 0;
  const int share = SPLIT ? (int)blockIdx.x % g.splits : 0, per_tile = SPLIT ? g.splits : CTAS;
  const int cta = (int)blockIdx.x / per_tile, ctas = (int)gridDim.x / per_tile;
  extern __shared__ unsigned char smem_raw[];
  const unsigned base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char *base_ptr = smem_raw + (base - smem_u32(smem_raw));
  const unsigned bars = base + L::BAR_OFF;
  auto full = [&](int s) { return bars + 8u * s; };
  auto empty = [&](int s) { return bars + 8u * (S + s); };
  auto chain_full = [&](int b) { return bars + 8u * (2 * S + b); };
  auto chain_empty = [&](int b) { return bars + 8u * (2 * S + CHAINS + b); };
  const unsigned done = bars + 8u * (2 * S + 2 * CHAINS);
  volatile unsigned *tmem_holder = reinterpret_cast<volatile unsigned *>(base_ptr + L::BAR_OFF + 120);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(base_ptr + L::BAR_OFF + 124);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int all_blocks = (g.k + 63) / 64, each = SPLIT ? (all_blocks + g.splits - 1) / g.splits : all_blocks;
  const int kb0 = min(all_blocks, share * each), kblocks = min(all_blocks, kb0 + each) - kb0;  // of this CTA
  auto place = [&](int tile, int &batch, int &mt, int &nt) {
    const int per = SYM ? g.m_tiles * (g.m_tiles + 1) / 2 : g.m_tiles * g.n_tiles;
    batch = tile / per;
    const int rest = tile - batch * per;
    if (SYM) {  // row mt has the tiles 0 .. mt
      mt = (int)((sqrtf(8.f * rest + 1.f) - 1.f) * 0.5f);
      while (mt * (mt + 1) / 2 > rest) --mt;
      while ((mt + 1) * (mt + 2) / 2 <= rest) ++mt;
      nt = rest - mt * (mt + 1) / 2;
    } else {
      mt = rest % g.m_tiles;
      nt = rest / g.m_tiles;
    }
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < CHAINS; ++b) {
      mbar_init(chain_full(b), 1);
      mbar_init(chain_empty(b), 8 * CTAS);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 0 && lane == 0)
    for (const CUtensorMap *map : {&map_ah, &map_al, &map_bh, &map_bl, &map_oh, &map_ol}) tma_prefetch_map(map);
  if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void *)tmem_holder)),
                   "r"(512u)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void *)tmem_holder)),
                   "r"(512u)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();  // both CTAs' barriers are there
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned tmem = *tmem_holder;
  pdl_wait();

  if (warp == 0) {
    int it = 0;
    bool ok = true;
    for (int tile = cta; tile < g.tiles && ok; tile += ctas) {
      int batch, mt, nt;
      place(tile, batch, mt, nt);
      for (int kb = 0; kb < kblocks; ++kb, ++it) {
        const int s = it % S;
        ok = mbar_wait_warp(empty(s), ((unsigned)(it / S) & 1u) ^ 1u, abort_flag, nullptr, 61);
        if (!ok) break;
        if (lane == 0) {
          const unsigned st = base + (unsigned)(s * L::STAGE);
          // (of a pair, the even one's barrier counts both CTAs' bytes)
          if (rank == 0) mbar_expect_tx(full(s), (unsigned)(CTAS * L::STAGE));
          const unsigned bar = PAIR ? cluster_map(full(s), 0) : full(s);
          auto load = [&](unsigned to, const CUtensorMap *map, bool mn, int r0) {
            const int k0 = (kb0 + kb) * 64;
            if (mn) {  // rows of k, two slabs of 64 columns
              ns_load<PAIR>(to, map, r0, k0, batch, bar);
              ns_load<PAIR>(to + 8192, map, r0 + 64, k0, batch, bar);
            } else {
              ns_load<PAIR>(to, map, k0, r0, batch, bar);
            }
          };
          const int m0 = mt * T + rank * 128, n0 = nt * T + rank * 128;
          load(st, &map_ah, A_MN, m0);
          load(st + L::TILE, &map_al, A_MN, m0);
          load(st + 2 * L::TILE, &map_bh, B_MN, n0);
          load(st + 3 * L::TILE, &map_bl, B_MN, n0);
        }
        __syncwarp();
      }
    }
    if (PAIR && *abort_flag) {  // copies in flight must land (only the even CTA's barriers know: a millisecond is ample)
      const unsigned long long limit = global_timer() + 1000000ull;
      while (global_timer() < limit) {}
    } else if (*abort_flag) {  // copies in flight must land before the shared memory goes away
      const unsigned long long limit = global_timer() + WAIT_LIMIT_NS;
      for (int j = it > S ? it - S : 0; j < it; ++j)
        while (!mbar_try_wait(full(j % S), (unsigned)(j / S) & 1u) && global_timer() < limit) {}
    }
  } else if (warp == 1) {
    constexpr unsigned idesc = (umma_idesc_f16(T) + (PAIR ? (unsigned)(TC_BM >> 4) << 24 : 0u)) |
                               (A_MN ? UMMA_A_MN_MAJOR : 0u) | (B_MN ? UMMA_B_MN_MAJOR : 0u);
    int it = 0;
    bool ok = true;
    for (int tile = rank == 0 ? cta : g.tiles; tile < g.tiles && ok; tile += ctas) {
      for (int kb = 0; kb < kblocks; ++kb, ++it) {
        const int s = it % S, buf = it % CHAINS;
        ok = mbar_wait_warp(full(s), (unsigned)(it / S) & 1u, abort_flag, nullptr, 63) &&
             mbar_wait_warp(chain_empty(buf), ((unsigned)(it / CHAINS) & 1u) ^ 1u, abort_flag, nullptr, 62);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (tc_elect()) {
          const unsigned st = base + (unsigned)(s * L::STAGE), d = tmem + (unsigned)(buf * T);
          const unsigned long long a0 = A_MN ? umma_desc_mn128(st, 8192u) : umma_desc_k128(st);
          const unsigned long long b0 = B_MN ? umma_desc_mn128(st + 2 * L::TILE, 8192u) : umma_desc_k128(st + 2 * L::TILE);
          auto a = [&](int part, int ks) { return a0 + (unsigned long long)(part * (L::TILE >> 4) + ks * (A_MN ? 2048 >> 4 : 2)); };
          auto b = [&](int part, int ks) { return b0 + (unsigned long long)(part * (L::TILE >> 4) + ks * (B_MN ? 2048 >> 4 : 2)); };
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            ns_mma<PAIR>(d, a(0, ks), b(1, ks), idesc, ks ? NS_ADD : NS_NEW);
            ns_mma<PAIR>(d, a(1, ks), b(0, ks), idesc, NS_ADD);
          }
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) ns_mma<PAIR>(d, a(0, ks), b(0, ks), idesc, ks ? NS_ADD : NS_SCALED);
          ns_commit<PAIR>(empty(s));
          ns_commit<PAIR>(chain_full(buf));
        }
        __syncwarp();
      }
    }
    if (!ok) {  // what was issued ends, within the limit, before the shared memory goes away
      if (tc_elect()) ns_commit<PAIR>(done);
      __syncwarp();
      const unsigned long long limit = global_timer() + WAIT_LIMIT_NS;
      while (!mbar_try_wait(done, 0u) && global_timer() < limit) {}
    }
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    unsigned char *patch = base_ptr + L::PATCH_OFF + (warp - 2) * L::PATCH;
    const unsigned patch_u = base + (unsigned)(L::PATCH_OFF + (warp - 2) * L::PATCH);
    int it = 0;
    bool ok = true;
    for (int tile = cta; tile < g.tiles; tile += ctas) {
      int batch, mt, nt;
      place(tile, batch, mt, nt);
      const float rho = g.rho[batch];
      const int row0 = mt * T + rank * 128 + q * 32;
      float acc[COLS];
      int ex, ea, eb;
      auto exponents = [&]() {
        ex = ns_exp_x(rho, g.step);
        ea = ns_exp_a(rho, g.step);
        eb = ns_exp_b(rho, g.step);
      };
      if (OP == GRAM || share > 0) {
        exponents();
#pragma unroll
        for (int j = 0; j < COLS; ++j) acc[j] = 0.f;
      } else {  // the added matrix, whole rows' 128 bytes at a time through the patch; all loads of 64 columns in flight
        if (lane == 0) bulk_wait_read<0>();
        __syncwarp();
#pragma unroll
        for (int c0 = 0; c0 < COLS; c0 += 64) {
          const int col0 = nt * T + half * COLS + c0;
          const long long from = ((long long)batch * g.m + row0) * g.ld + col0 + (lane & 7) * 8;
          const bool in = col0 + (lane & 7) * 8 < g.n;
          uint4 u[2][8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (lane >> 3);
            const bool there = in && row0 + r < g.m;
            u[0][i] = there ? *reinterpret_cast<const uint4 *>(g.add.hi + from + r * g.ld) : make_uint4(0u, 0u, 0u, 0u);
            u[1][i] = there ? *reinterpret_cast<const uint4 *>(g.add.lo + from + r * g.ld) : make_uint4(0u, 0u, 0u, 0u);
          }
          if (c0 == 0) exponents();
          const float f_add = OP == POLY ? NS_B / NS_C * ns_pow2(ea) : NS_A * ns_pow2(eb);
#pragma unroll
          for (int lo = 0; lo < 2; ++lo) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = i * 4 + (lane >> 3);
              *reinterpret_cast<uint4 *>(patch + r * 128 + (((lane & 7) ^ (r & 7)) << 4)) = u[lo][i];
            }
            __syncwarp();
            const float f = lo ? f_add / 2048.f : f_add;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint4 v = *reinterpret_cast<const uint4 *>(patch + lane * 128 + ((i ^ (lane & 7)) << 4));
              const __half2 *z = reinterpret_cast<const __half2 *>(&v);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float2 w = __half22float2(z[j]);
                const int at = c0 + i * 8 + 2 * j;
                acc[at] = lo ? fmaf(w.x, f, acc[at]) : w.x * f;
                acc[at + 1] = lo ? fmaf(w.y, f, acc[at + 1]) : w.y * f;
              }
            }
            __syncwarp();
          }
        }
      }
      // acc = the product times 2^(sum of the operands' exponents), which may reach 200: two factors
      const int e_in = OP == GRAM ? 2 * ex : OP == POLY ? 2 * ea : eb + ex;
      const int e_out = OP == GRAM ? ea : OP == POLY ? eb : ns_exp_x(rho, g.step + 1);
      const float f2 = ns_pow2(e_out - (e_in - e_in / 2));
      for (int kb = 0; kb < kblocks && ok; ++kb, ++it) {
        const int buf = it % CHAINS;
        ok = mbar_wait_warp(chain_full(buf), (unsigned)(it / CHAINS) & 1u, abort_flag, nullptr, 64);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
        for (int c0 = 0; c0 < COLS; c0 += 32) {
          unsigned r[32];
          tc_ld32(tmem + ((unsigned)(q * 32) << 16) + (unsigned)(buf * T + half * COLS + c0), r);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[c0 + j] += __uint_as_float(r[j]);
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIR)
            asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_map(chain_empty(buf), 0))
                         : "memory");
          else mbar_arrive(chain_empty(buf));
        }
      }
      const float f1 = ok ? (OP == POLY ? NS_C : 1.f) * ns_pow2(-(e_in / 2)) : NAN;
      if constexpr (SPLIT) {  // every product has been read: this range's sums may lie over the stages
        float *sums = reinterpret_cast<float *>(base_ptr) + (q * 32 + lane) * NS_LD + half * COLS;
#pragma unroll
        for (int j = 0; j < COLS; j += 4)
          *reinterpret_cast<float4 *>(sums + j) = make_float4(acc[j] * f1 * f2, acc[j + 1] * f1 * f2, acc[j + 2] * f1 * f2, acc[j + 3] * f1 * f2);
        break;
      } else {
#pragma unroll
      for (int c0 = 0; c0 < COLS; c0 += 32) {
        const int col = nt * T + half * COLS + c0;
        if (col >= g.n || row0 >= g.m) continue;
        unsigned h[16], l[16];
#pragma unroll
        for (int j = 0; j < 32; j += 2) ns_split2(acc[c0 + j] * f1 * f2, acc[c0 + j + 1] * f1 * f2, h[j >> 1], l[j >> 1]);
        if (lane == 0) bulk_wait_read<0>();
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int to = lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4);
          *reinterpret_cast<uint4 *>(patch + to) = make_uint4(h[4 * j], h[4 * j + 1], h[4 * j + 2], h[4 * j + 3]);
          *reinterpret_cast<uint4 *>(patch + 2048 + to) = make_uint4(l[4 * j], l[4 * j + 1], l[4 * j + 2], l[4 * j + 3]);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          tma_store_4d(&map_oh, patch_u, col, 0, row0, batch);
          tma_store_4d(&map_ol, patch_u + 2048, col, 0, row0, batch);
        }
        if (!SYM || mt == nt) continue;
        if (lane == 0) bulk_wait_read<0>();
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 32; ++j) {  // the same turned: row j is column col + j
          const int to = j * 64 + (((lane >> 3) ^ ((j >> 1) & 3)) << 4) + (lane & 7) * 2;
          *reinterpret_cast<unsigned short *>(patch + to) = (unsigned short)(h[j >> 1] >> (16 * (j & 1)));
          *reinterpret_cast<unsigned short *>(patch + 2048 + to) = (unsigned short)(l[j >> 1] >> (16 * (j & 1)));
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          tma_store_4d(&map_oh, patch_u, row0, 0, col, batch);
          tma_store_4d(&map_ol, patch_u + 2048, row0, 0, col, batch);
        }
      }
      }
    }
    if (lane == 0) bulk_wait_all();  // the stores are part of the grid's results
  }
  if constexpr (SPLIT) {  // one tile, its ranges of k over the CTAs of the cluster: each stores a share of the rows
    __syncwarp();
    cluster_sync_all();
    int batch, mt, nt;
    place(cta, batch, mt, nt);
    const int rows = 128 / g.splits, r0 = share * rows;
    float *whole = reinterpret_cast<float *>(base_ptr + 128 * NS_LD * 4);  // [rows][NS_LD]
    for (int e = threadIdx.x; e < rows * 32; e += NS_THREADS) {
      const int r = e / 32, c = e % 32 * 4;
      const unsigned from = base + (unsigned)((r0 + r) * NS_LD + c) * 4u;
      float4 v = ld_cluster_f4(cluster_map(from, 0u));
      for (int i = 1; i < g.splits; ++i) {
        const float4 w = ld_cluster_f4(cluster_map(from, (unsigned)i));
        v = make_float4(v.x + w.x, v.y + w.y, v.z + w.z, v.w + w.w);
      }
      *reinterpret_cast<float4 *>(whole + r * NS_LD + c) = v;
    }
    __syncthreads();
    auto store8 = [&](int row, int col, const float (&v)[8]) {  // columns col .. col + 7 of a row of the result
      unsigned h[4], l[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) ns_split2(v[2 * j], v[2 * j + 1], h[j], l[j]);
      const long long to = ((long long)batch * g.m + row) * g.ld + col;
      *reinterpret_cast<uint4 *>(g.out.hi + to) = make_uint4(h[0], h[1], h[2], h[3]);
      *reinterpret_cast<uint4 *>(g.out.lo + to) = make_uint4(l[0], l[1], l[2], l[3]);
    };
    for (int e = threadIdx.x; e < rows * 16; e += NS_THREADS) {
      const int r = e / 16, c = e % 16 * 8, row = mt * 128 + r0 + r, col = nt * 128 + c;
      if (row >= g.m || col >= g.n) continue;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = whole[r * NS_LD + c + j];
      store8(row, col, v);
    }
    if (SYM && mt != nt) {
      for (int e = threadIdx.x; e < rows * 16; e += NS_THREADS) {  // a column, eight rows (those behind the matrix are its padding)
        const int c = e % 128, r = e / 128 * 8, row = nt * 128 + c, col = mt * 128 + r0 + r;
        if (row >= g.n || col >= g.m) continue;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = whole[(r + j) * NS_LD + c];
        store8(row, col, v);
      }
    }
    __syncwarp();
    cluster_sync_all();  // no peer reads these sums any more
  }
  __syncwarp();
  pdl_launch_dependents();  // here and not at the start: a step of 256 x 256 takes 23.9 us so, 26.7 with waiting CTAs around
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();  // nothing of the pair's is on its way to the other CTA
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

struct Operand {
  Pair p;
  long long rows, cols, ld;
};

CUtensorMap ns_map(const __half *p, const Operand &o, long long count, bool mn, bool result = false) {
  CUtensorMap map;
  const unsigned long long extent[4] = {(unsigned long long)o.cols, 1, (unsigned long long)o.rows, (unsigned long long)count};
  const unsigned long long strides[3] = {16, (unsigned long long)o.ld * 2, (unsigned long long)(o.rows * o.ld) * 2};
  if (result) tc_make_map_heads(&map, p, extent, strides, 32, 32);
  else tc_make_map_heads(&map, p, extent, strides, mn ? 64 : 128);
  return map;
}

template <NsOp OP, bool A_MN, bool B_MN, bool PAIR, bool SPLIT>
void launch_product(const Operand &a, const Operand &b, const Operand &out, NsProduct g, long long count, cudaStream_t st) {
  constexpr int CTAS = PAIR ? 2 : 1, T = 128 * CTAS;
  g.m_tiles = (g.m + T - 1) / T;
  g.n_tiles = (g.n + T - 1) / T;
  const long long per = OP == APPLY ? (long long)g.m_tiles * g.n_tiles : (long long)g.m_tiles * (g.m_tiles + 1) / 2;
  g.tiles = (int)(per * count);  // (in range: checked before the call's first kernel)
  using L = NsSmem;
  static SharedMemoryOnce once;
  once.set(ns_product_kernel<OP, A_MN, B_MN, PAIR, SPLIT>, L::TOTAL);
  const int per_tile = SPLIT ? g.splits : CTAS, ctas = SPLIT || g.tiles < 148 / CTAS ? g.tiles : 148 / CTAS;
  launch_pdl_cluster_x(ns_product_kernel<OP, A_MN, B_MN, PAIR, SPLIT>, dim3((unsigned)(ctas * per_tile)), dim3(NS_THREADS), L::TOTAL, st,
                       true, (unsigned)per_tile, ns_map(a.p.hi, a, count, A_MN), ns_map(a.p.lo, a, count, A_MN), ns_map(b.p.hi, b, count, B_MN),
                       ns_map(b.p.lo, b, count, B_MN), ns_map(out.p.hi, out, count, false, true),
                       ns_map(out.p.lo, out, count, false, true), g);
}

template <NsOp OP, bool A_MN, bool B_MN>
void product(const Operand &a, const Operand &b, const Operand &out, int k, const Pair &add, int step, const float *rho,
             long long count, cudaStream_t st) {
  NsProduct g{};
  g.add = add;
  g.out = out.p;
  g.splits = 1;
  g.ld = out.ld;
  g.m = (int)out.rows;
  g.n = (int)out.cols;
  g.k = k;
  g.step = step;
  g.rho = rho;
  // us of the longest CTA: a turn's blocks of 64 k and what surrounds them, and a launch. A CTA's 64 KB of operands a block come at
  // 50 bytes a clock (0.69 us, of which 0.4 are products), a little slower with all SMs at it; a pair's CTAs take the same for twice
  // the result (1.07 us, the tensor pipe 0.8) and longer before and behind it. Four matrices of 4096 x 1024, a step: A 60 us by single
  // CTAs, 80 by pairs (80 of 148 SMs); X 116 and 103. Six of 512 x 2048: X 32 and 39.
  const double kb = (k + 63) / 64;
  auto turns = [&](long long t, long long at_once, double &busy) {
    const long long mt = (g.m + t - 1) / t, nt = (g.n + t - 1) / t, tiles = (OP == APPLY ? mt * nt : mt * (mt + 1) / 2) * count;
    busy = tiles < at_once ? (double)tiles / at_once : 1.0;
    return (double)((tiles + at_once - 1) / at_once);
  };
  double busy = 0;
  const double pair = turns(256, 74, busy) * (kb * 1.07 + 9) + 3.5;
  const double one = turns(128, 148, busy) * (kb * (busy > 0.8 ? 0.86 * busy : 0.69) + 2.5) + 2.5;
  // Few tiles: a tile's k over the CTAs of a cluster, joined over distributed shared memory.
  const long long mt = (g.m + 127) / 128, nt = (g.n + 127) / 128, tiles = (OP == APPLY ? mt * nt : mt * (mt + 1) / 2) * count;
  const int *fit = tc_cluster_capacity();
  double least = one < pair ? one : pair;
  for (int s = 2; s <= 8; s *= 2) {
    if (tiles * s > 148 || tiles > fit[s] || kb < s) break;
    const double t = ceil(kb / s) * 0.69 + NS_SPLIT + 2.5 + 2.5;
    if (t < least) {
      least = t;
      g.splits = s;
    }
  }
  if (g.splits > 1) launch_product<OP, A_MN, B_MN, false, true>(a, b, out, g, count, st);
  else if (pair < one) launch_product<OP, A_MN, B_MN, true, false>(a, b, out, g, count, st);
  else launch_product<OP, A_MN, B_MN, false, false>(a, b, out, g, count, st);
}

bool rows16(const MatView &v) {
  if (v.cs != 4 || v.rs % 16 || reinterpret_cast<uintptr_t>(v.data) % 16) return false;
  for (int i = 0; i < v.nb; ++i)
    if (v.bs[i] % 16) return false;
  return true;
}

size_t up(size_t bytes) { return (bytes + 255) / 256 * 256; }

// The workspace's parts; its size.
size_t ns_layout(long long count, long long m, long long n, char *p, NsWork *w) {
  const long long small = m < n ? m : n;
  const long long ldx = (n + 7) / 8 * 8, ldp = (small + 7) / 8 * 8;
  char *const begin = p;
  auto take = [&](size_t bytes) {
    char *at = p;
    p += up(bytes);
    return at;
  };
  NsWork k;
  k.ldx = ldx;
  k.ldp = ldp;
  k.parts = reinterpret_cast<double *>(take((size_t)count * NS_PARTS * 8));
  k.rho = reinterpret_cast<float *>(take((size_t)count * 4));
  for (Pair *x : {&k.x[0], &k.x[1]}) {
    x->hi = reinterpret_cast<__half *>(take((size_t)count * m * ldx * 2));
    x->lo = reinterpret_cast<__half *>(take((size_t)count * m * ldx * 2));
  }
  for (Pair *x : {&k.a, &k.b}) {
    x->hi = reinterpret_cast<__half *>(take((size_t)count * small * ldp * 2));
    x->lo = reinterpret_cast<__half *>(take((size_t)count * small * ldp * 2));
  }
  if (w) *w = k;
  return (size_t)(p - begin);
}

}  // namespace

size_t muon_workspace_bytes(long long count, long long m, long long n) { return ns_layout(count, m, n, nullptr, nullptr); }

void launch_muon(const MuonStep &g, void *workspace, cudaStream_t st) {
  const long long m = g.grads.rows, n = g.grads.cols, count = g.grads.batch;
  if (muon_small_supports(m, n)) return launch_muon_small(g, st);
  const bool tall = m > n;
  const int p = (int)(tall ? n : m);
  NsWork w;
  ns_layout(count, m, n, static_cast<char *>(workspace), &w);
  const unsigned vec = (rows16(g.grads) ? VEC_G : 0) | (g.step && rows16(g.momentum) ? VEC_M : 0) | (rows16(g.params) ? VEC_P : 0);
  const long long quads = m * ((n + 3) / 4), blocks = (quads + 255) / 256;
  // as many blocks of a matrix as fill the chip together with the others', four groups to a thread where there are more
  const long long fill = (148 * 8 + count - 1) / count, each = blocks < fill ? blocks : fill;
  const unsigned parts = (unsigned)(each < NS_PARTS ? each : NS_PARTS);
  const dim3 grid(parts, (unsigned)count), wide((unsigned)each, (unsigned)count);
  auto dense = [&](const MatView &v) { return v.cs == 4 && v.rs == 4 * n; };
  const bool flat = n % 4 == 0 && w.ldx == n && vec == (unsigned)(VEC_G | (g.step ? VEC_M : 0) | VEC_P) && dense(g.grads) &&
                    dense(g.params) && (!g.step || dense(g.momentum));
  launch_pdl(flat ? muon_begin_kernel<true> : muon_begin_kernel<false>, grid, dim3(256), 0, st, true, g, w, vec);
  launch_pdl(flat ? muon_pair_kernel<true> : muon_pair_kernel<false>, wide, dim3(256), 0, st, true, g, w, vec, (int)parts);
  for (int i = 0; i < g.steps; ++i) {
    const Operand x{w.x[i & 1], m, n, w.ldx}, y{w.x[(i + 1) & 1], m, n, w.ldx}, a{w.a, p, p, w.ldp}, b{w.b, p, p, w.ldp};
    if (tall) product<GRAM, true, true>(x, x, a, (int)m, Pair{}, i, w.rho, count, st);
    else product<GRAM, false, false>(x, x, a, (int)n, Pair{}, i, w.rho, count, st);
    product<POLY, false, false>(a, a, b, p, a.p, i, w.rho, count, st);
    if (tall) product<APPLY, false, false>(x, b, y, p, x.p, i, w.rho, count, st);
    else product<APPLY, false, true>(b, x, y, p, x.p, i, w.rho, count, st);
  }
  const float rate = g.lr * sqrtf(m > n ? (float)m / (float)n : 1.f);
  launch_pdl(flat ? muon_end_kernel<true> : muon_end_kernel<false>, wide, dim3(256), 0, st, true, g, w, vec, 1.f - g.lr * g.weight_decay,
             rate);
}

}  // namespace lb

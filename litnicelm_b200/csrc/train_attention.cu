// Attention with its backward pass for training: bfloat16 operands that the tensor-core kernels cannot address (any sizes and
// strides), 32-bit arithmetic throughout:
//   forward   s_ij = scale q_i . k_j,  lse_i = log sum_j exp s_ij,  out_i = sum_j exp(s_ij - lse_i) v_j
//   backward  p_ij = exp(s_ij - lse_i) again from q, k and lse, delta_i = dout_i . out_i,
//             ds_ij = scale p_ij (dout_i . v_j - delta_i),
//             dq_i = sum_j ds_ij k_j,  dk_j = sum_i ds_ij q_i,  dv_j = sum_i p_ij dout_i
// over the keys j that row i sees; key heads shared by query heads receive the sum over those. A row that sees no key has
// out 0, lse -infinity and no part in any gradient.
//
// Tiles of 64 x 64 by 128 threads, 8 x 4 scores each (rows 8 apart, columns 16 apart: 8 + 8 wavefronts of shared memory for 128
// fused multiply-adds a warp), one pass over the keys with a running maximum and sum. Two kernels for the gradients, one by rows
// (dq) and one by keys (dk, dv), so that no sum depends on the order in which blocks finish; the scores are computed in both.
// Bound: the FMA pipe: 2 streams of 1024 rows, 8 heads of 64, causal, 240 us forward and 620 backward (as rows that TMA can address 21 and
// 36 on the tensor cores).
#include "train_ops.cuh"

#include <cuda_bf16.h>

namespace lb {

namespace {

typedef __nv_bfloat16 bf16;

constexpr int TA_B = 64, TA_THREADS = 128;
constexpr float TA_LOG2E = 1.4426950408889634f;

// Four consecutive elements of a row, of which `count` exist.
__device__ __forceinline__ float4 load4(const bf16 *p, long long c, int count, bool vec) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (vec && count >= 4) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&u.x));
    const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&u.y));
    return make_float4(a.x, a.y, b.x, b.y);
  }
  if (count > 0) v.x = __bfloat162float(p[0]);
  if (count > 1) v.y = __bfloat162float(p[c]);
  if (count > 2) v.z = __bfloat162float(p[2 * c]);
  if (count > 3) v.w = __bfloat162float(p[3 * c]);
  return v;
}

struct TaArgs {
  TrainAttention a;
  float *delta;
  int tiles;        // of 64 rows (or keys) per head
  unsigned vec;     // bit per view: rows can be read four elements at a time
};
enum { VQ = 1, VK = 2, VV = 4, VDO = 8, VO = 16 };

// Rows r0 .. r0 + 63 of a head into shared memory, those from `end` on, or before `begin`, and the columns behind dim as zeros.
template <int D>
__device__ __forceinline__ void load_tile(float *to, const HeadView &x, long long base, int r0, int end, int dim, bool vec, int begin = 0) {
  constexpr int LD = D + 4, Q = D / 4;
  const bf16 *p = reinterpret_cast<const bf16 *>(x.p) + base;
#pragma unroll 4
  for (int e = threadIdx.x; e < TA_B * Q; e += TA_THREADS) {
    const int r = e / Q, c = e % Q * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r0 + r >= begin && r0 + r < end) v = load4(p + (long long)(r0 + r) * x.r + c * x.c, x.c, dim - c, vec);
    *reinterpret_cast<float4 *>(to + r * LD + c) = v;
  }
}

// s[i][j] = rows (i * 8 + ty) of a . rows (j * 16 + tx) of b
template <int D>
__device__ __forceinline__ void tile_dot(const float *a, const float *b, float (&s)[8][4]) {
  constexpr int LD = D + 4;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 2
  for (int c = 0; c < D; c += 4) {
    float4 y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4 *>(b + (j * 16 + tx) * LD + c);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 x = *reinterpret_cast<const float4 *>(a + (i * 8 + ty) * LD + c);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        s[i][j] = fmaf(x.w, y[j].w, fmaf(x.z, y[j].z, fmaf(x.y, y[j].y, fmaf(x.x, y[j].x, s[i][j]))));
    }
  }
}

constexpr int TA_LP = TA_B + 4;

// acc[i][..] += sum over t of w[i * 8 + ty][t] b[t][columns of this thread]
template <int D>
__device__ __forceinline__ void tile_mul(const float *w, const float *b, float (&acc)[8][D / 16]) {
  constexpr int LD = D + 4, W = D >= 64 ? 4 : 2;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll 1
  for (int t = 0; t < TA_B; t += 4) {
    float4 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const float4 *>(w + (i * 8 + ty) * TA_LP + t);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int c = 0; c < D / 16; c += W) {
        float y[W];
        const float *p = b + (t + u) * LD + (c / W) * 64 + tx * W;
        if constexpr (W == 4) {
          const float4 v = *reinterpret_cast<const float4 *>(p);
          y[0] = v.x; y[1] = v.y; y[2] = v.z; y[3] = v.w;
        } else {
          const float2 v = *reinterpret_cast<const float2 *>(p);
          y[0] = v.x; y[1] = v.y;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float f = u == 0 ? x[i].x : u == 1 ? x[i].y : u == 2 ? x[i].z : x[i].w;
#pragma unroll
          for (int e = 0; e < W; ++e) acc[i][c + e] = fmaf(f, y[e], acc[i][c + e]);
        }
      }
    }
  }
}

template <int D>
__device__ __forceinline__ void store_tile(const HeadView &x, long long base, int r0, int end, int dim, float (&acc)[8][D / 16],
                                           const float (&factor)[8]) {
  constexpr int W = D >= 64 ? 4 : 2;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  bf16 *p = reinterpret_cast<bf16 *>(x.p) + base;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + i * 8 + ty;
    if (r >= end) continue;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      const int col = (c / W) * 64 + tx * W + c % W;
      if (col < dim) p[(long long)r * x.r + col * x.c] = __float2bfloat16_rn(acc[i][c] * factor[i]);
    }
  }
}

__device__ __forceinline__ float row_max16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float row_sum16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Which tile, head and stream a block has; the tiles with the most keys first.
struct TaPlace {
  int tile, head, stream, keys;
};
__device__ __forceinline__ TaPlace ta_place(const TaArgs &g, int heads, bool last_first) {
  const long long b = blockIdx.x;
  const long long each = (long long)heads * g.a.streams;
  const int t = (int)(b / each), rest = (int)(b - t * each);
  TaPlace p;
  p.tile = last_first ? g.tiles - 1 - t : t;
  p.stream = rest / heads;
  p.head = rest - p.stream * heads;
  p.keys = g.a.seen;
  if (g.a.lengths) p.keys = max(0, min(g.a.seen, g.a.lengths[p.stream]));
  return p;
}

template <int D>
__global__ void __launch_bounds__(TA_THREADS)
train_attention_forward_kernel(const __grid_constant__ TaArgs g) {
  constexpr int LD = D + 4;
  extern __shared__ float sm[];
  float *sq = sm, *sk = sq + TA_B * LD, *sv = sk + TA_B * LD, *sp = sv + TA_B * LD;
  const TrainAttention &a = g.a;
  const TaPlace at = ta_place(g, a.heads, a.causal != 0);
  const TrainSpan span{a.first, a.window, a.causal};
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int r0 = at.tile * TA_B, r1 = min(r0 + TA_B, a.n), kh = at.head / (a.heads / a.groups);
  const long long qb = at.stream * a.q.s + at.head * a.q.h, kb = at.stream * a.k.s + kh * a.k.h,
                  vb = at.stream * a.v.s + kh * a.v.h;
  load_tile<D>(sq, a.q, qb, r0, a.n, a.dim, g.vec & VQ);
  const int lo = span.lo(r0) / TA_B * TA_B, end = span.end(r1 - 1, at.keys);
  float o[8][D / 16], m[8], l[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) o[i][c] = 0.f;
  }
  const float f = a.scale * TA_LOG2E;
  for (int j0 = lo; j0 < end; j0 += TA_B) {
    __syncthreads();
    load_tile<D>(sk, a.k, kb, j0, at.keys, a.dim, g.vec & VK, span.lo(r0));
    load_tile<D>(sv, a.v, vb, j0, at.keys, a.dim, g.vec & VV, span.lo(r0));
    __syncthreads();
    float s[8][4];
    tile_dot<D>(sq, sk, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = r0 + i * 8 + ty, first = span.lo(row), last = span.end(row, at.keys);
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = j0 + j * 16 + tx;
        s[i][j] = key >= first && key < last ? __fmul_rn(s[i][j], f) : -INFINITY;  // (rounded, or the difference from m is not)
        top = fmaxf(top, s[i][j]);
      }
      top = fmaxf(m[i], row_max16(top));
      const float base = top == -INFINITY ? 0.f : top;
      const float keep = exp2f(m[i] - base);
      m[i] = top;
      l[i] *= keep;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) o[i][c] *= keep;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = exp2f(s[i][j] - base);
        l[i] += p;
        sp[(i * 8 + ty) * TA_LP + j * 16 + tx] = p;
      }
    }
    __syncthreads();
    tile_mul<D>(sp, sv, o);
  }
  float inv[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float total = row_sum16(l[i]);
    inv[i] = total > 0.f ? 1.0f / total : (total == 0.f ? 0.f : total);  // a sum that is not a number stays that
    const int row = r0 + i * 8 + ty;
    if (tx == 0 && row < a.n)
      a.lse[((long long)at.stream * a.heads + at.head) * a.n + row] = total == 0.f ? -INFINITY : m[i] / TA_LOG2E + logf(total);
  }
  store_tile<D>(a.out, at.stream * a.out.s + at.head * a.out.h, r0, a.n, a.dim, o, inv);
}

// A row by LANES lanes, eight elements each.
template <int LANES>
__global__ void __launch_bounds__(256) train_delta_kernel(const __grid_constant__ TaArgs g) {
  pdl_launch_dependents();
  const TrainAttention &a = g.a;
  // rows in the order of memory as layers leave it, [streams, n, heads]: neighbours of a warp read on
  const long long rows = (long long)a.streams * a.heads * a.n, mine = blockIdx.x * (256LL / LANES) + threadIdx.x / LANES;
  const long long at = mine < rows ? mine : rows - 1;
  const int lane = threadIdx.x % LANES, c = lane * 8;
  const long long si = div_index(at, a.heads), s = div_index(si, a.n);
  const int h = (int)(at - si * a.heads), i = (int)(si - s * a.n);
  const bf16 *x = reinterpret_cast<const bf16 *>(a.out.p) + s * a.out.s + (long long)i * a.out.r + h * a.out.h + c * a.out.c;
  const bf16 *y = reinterpret_cast<const bf16 *>(a.dout.p) + s * a.dout.s + (long long)i * a.dout.r + h * a.dout.h + c * a.dout.c;
  float t = 0.f;
#pragma unroll
  for (int e = 0; e < 8; e += 4) {
    const float4 u = load4(x + e * a.out.c, a.out.c, a.dim - c - e, g.vec & VO);
    const float4 v = load4(y + e * a.dout.c, a.dout.c, a.dim - c - e, g.vec & VDO);
    t = fmaf(u.x, v.x, fmaf(u.y, v.y, fmaf(u.z, v.z, fmaf(u.w, v.w, t))));
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if (lane == 0 && mine < rows) g.delta[(s * a.heads + h) * a.n + i] = t;
}

template <int D>
__global__ void __launch_bounds__(TA_THREADS)
train_attention_dq_kernel(const __grid_constant__ TaArgs g) {
  constexpr int LD = D + 4;
  extern __shared__ float sm[];
  float *sq = sm, *sdo = sq + TA_B * LD, *sk = sdo + TA_B * LD, *sv = sk + TA_B * LD, *sp = sv + TA_B * LD;
  const TrainAttention &a = g.a;
  const TaPlace at = ta_place(g, a.heads, a.causal != 0);
  const TrainSpan span{a.first, a.window, a.causal};
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int r0 = at.tile * TA_B, r1 = min(r0 + TA_B, a.n), kh = at.head / (a.heads / a.groups);
  const long long qb = at.stream * a.q.s + at.head * a.q.h, kb = at.stream * a.k.s + kh * a.k.h,
                  vb = at.stream * a.v.s + kh * a.v.h, db = at.stream * a.dout.s + at.head * a.dout.h;
  load_tile<D>(sq, a.q, qb, r0, a.n, a.dim, g.vec & VQ);
  load_tile<D>(sdo, a.dout, db, r0, a.n, a.dim, g.vec & VDO);
  float lse[8], delta[8], acc[8][D / 16], one[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = r0 + i * 8 + ty;
    const long long x = ((long long)at.stream * a.heads + at.head) * a.n + row;
    lse[i] = row < a.n ? a.lse[x] * TA_LOG2E : 0.f;
    delta[i] = row < a.n ? g.delta[x] : 0.f;
    one[i] = a.scale;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) acc[i][c] = 0.f;
  }
  const int lo = span.lo(r0) / TA_B * TA_B, end = span.end(r1 - 1, at.keys);
  const float f = a.scale * TA_LOG2E;
  for (int j0 = lo; j0 < end; j0 += TA_B) {
    __syncthreads();
    load_tile<D>(sk, a.k, kb, j0, at.keys, a.dim, g.vec & VK, span.lo(r0));
    load_tile<D>(sv, a.v, vb, j0, at.keys, a.dim, g.vec & VV, span.lo(r0));
    __syncthreads();
    float s[8][4], dp[8][4];
    tile_dot<D>(sq, sk, s);
    tile_dot<D>(sdo, sv, dp);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = r0 + i * 8 + ty, first = span.lo(row), last = span.end(row, at.keys);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = j0 + j * 16 + tx;
        const float p = exp2f(fmaf(s[i][j], f, -lse[i]));
        sp[(i * 8 + ty) * TA_LP + j * 16 + tx] = row < a.n && key >= first && key < last ? p * (dp[i][j] - delta[i]) : 0.f;
      }
    }
    __syncthreads();
    tile_mul<D>(sp, sk, acc);
  }
  store_tile<D>(a.dq, at.stream * a.dq.s + at.head * a.dq.h, r0, a.n, a.dim, acc, one);
}

template <int D>
__global__ void __launch_bounds__(TA_THREADS)
train_attention_dkv_kernel(const __grid_constant__ TaArgs g) {
  constexpr int LD = D + 4;
  extern __shared__ float sm[];
  float *sk = sm, *sv = sk + TA_B * LD, *sq = sv + TA_B * LD, *sdo = sq + TA_B * LD, *sp = sdo + TA_B * LD;
  const TrainAttention &a = g.a;
  const TaPlace at = ta_place(g, a.groups, false);
  const TrainSpan span{a.first, a.window, a.causal};
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int j0 = at.tile * TA_B, share = a.heads / a.groups;
  const long long kb = at.stream * a.k.s + at.head * a.k.h, vb = at.stream * a.v.s + at.head * a.v.h;
  float dk[8][D / 16], dv[8][D / 16], one[8], scales[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    one[i] = 1.f;
    scales[i] = a.scale;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) dk[i][c] = dv[i][c] = 0.f;
  }
  if (j0 < at.keys) {
    load_tile<D>(sk, a.k, kb, j0, at.keys, a.dim, g.vec & VK);
    load_tile<D>(sv, a.v, vb, j0, at.keys, a.dim, g.vec & VV);
    // rows that see a key of this tile
    const int j1 = min(j0 + TA_B, at.keys);
    const int lo = a.causal ? max(0, j0 - a.first) / TA_B * TA_B : 0;
    const long long past = a.window > 0 ? (long long)j1 - 1 + a.window - a.first : a.n;
    const int end = past < a.n ? (int)max(past, 0LL) : a.n;
    const int live = span.rows_end(a.n, at.keys);  // what rows that see no key hold must not meet their weights of zero
    const float f = a.scale * TA_LOG2E;
    for (int h = at.head * share; h < (at.head + 1) * share; ++h) {
      const long long qb = at.stream * a.q.s + h * a.q.h, db = at.stream * a.dout.s + h * a.dout.h;
      const long long stat = ((long long)at.stream * a.heads + h) * a.n;
      for (int r0 = lo; r0 < end; r0 += TA_B) {
        __syncthreads();
        load_tile<D>(sq, a.q, qb, r0, live, a.dim, g.vec & VQ);
        load_tile<D>(sdo, a.dout, db, r0, live, a.dim, g.vec & VDO);
        __syncthreads();
        float s[8][4];
        tile_dot<D>(sk, sq, s);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = r0 + j * 16 + tx, first = span.lo(row), last = span.end(row, at.keys);
          const float lse = row < a.n ? a.lse[stat + row] * TA_LOG2E : 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int key = j0 + i * 8 + ty;
            s[i][j] = row < a.n && key >= first && key < last ? exp2f(fmaf(s[i][j], f, -lse)) : 0.f;
            sp[(i * 8 + ty) * TA_LP + j * 16 + tx] = s[i][j];
          }
        }
        __syncthreads();
        tile_mul<D>(sp, sdo, dv);
        float dp[8][4];
        tile_dot<D>(sv, sdo, dp);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = r0 + j * 16 + tx;
          const float delta = row < a.n ? g.delta[stat + row] : 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            sp[(i * 8 + ty) * TA_LP + j * 16 + tx] = s[i][j] != 0.f ? s[i][j] * (dp[i][j] - delta) : 0.f;
        }
        __syncthreads();
        tile_mul<D>(sp, sq, dk);
      }
    }
  }
  store_tile<D>(a.dk, at.stream * a.dk.s + at.head * a.dk.h, j0, a.m, a.dim, dk, scales);
  store_tile<D>(a.dv, at.stream * a.dv.s + at.head * a.dv.h, j0, a.m, a.dim, dv, one);
}

bool rows_vec(const HeadView &x) {
  return x.c == 1 && x.r % 4 == 0 && x.h % 4 == 0 && x.s % 4 == 0 && reinterpret_cast<uintptr_t>(x.p) % 8 == 0;
}

TaArgs ta_args(const TrainAttention &a, float *delta, int rows) {
  TaArgs g{};
  g.a = a;
  g.delta = delta;
  g.tiles = (rows + TA_B - 1) / TA_B;
  g.vec = (rows_vec(a.q) ? VQ : 0) | (rows_vec(a.k) ? VK : 0) | (rows_vec(a.v) ? VV : 0) |
          (a.dout.p && rows_vec(a.dout) ? VDO : 0) | (a.out.p && rows_vec(a.out) ? VO : 0);
  return g;
}

unsigned ta_grid(const TaArgs &g, int heads) {
  const long long blocks = (long long)g.tiles * heads * g.a.streams;
  if (blocks > 0x7fffffffLL) throw std::invalid_argument("attention: too many rows, heads and streams for one call");
  return (unsigned)blocks;
}

template <typename F>
void launch(F kernel, const TaArgs &g, unsigned grid, int d, int tiles, cudaStream_t st) {
  const size_t smem = sizeof(float) * ((size_t)tiles * TA_B * (d + 4) + TA_B * TA_LP);
  LB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  kernel<<<grid, TA_THREADS, smem, st>>>(g);
  LB_LAUNCH_CHECK();
}

template <int D>
void forward(const TaArgs &g, cudaStream_t st) {
  launch(train_attention_forward_kernel<D>, g, ta_grid(g, g.a.heads), D, 3, st);
}
template <int D>
void backward(const TrainAttention &a, float *delta, cudaStream_t st) {
  const TaArgs gk = ta_args(a, delta, a.m), gq = ta_args(a, delta, a.n);
  launch(train_attention_dkv_kernel<D>, gk, ta_grid(gk, a.groups), D, 4, st);
  launch(train_attention_dq_kernel<D>, gq, ta_grid(gq, a.heads), D, 4, st);
}

template <int LANES>
void launch_delta(const TrainAttention &a, float *delta, cudaStream_t st) {
  const TaArgs g = ta_args(a, delta, a.n);
  const long long blocks = ((long long)a.streams * a.heads * a.n + 256 / LANES - 1) / (256 / LANES);
  if (blocks > 0x7fffffffLL) throw std::invalid_argument("attention: too many rows, heads and streams for one call");
  train_delta_kernel<LANES><<<(unsigned)blocks, 256, 0, st>>>(g);
  LB_LAUNCH_CHECK();
}

}  // namespace

void launch_train_attention_forward(const TrainAttention &a, void *work, cudaStream_t st) {
  if (!a.bf16) return launch_train_attention_forward_f32(a, work, st);
  if (train_attention_tc_supports(a, false)) return launch_train_attention_forward_tc(a, st);
  const TaArgs g = ta_args(a, nullptr, a.n);
  if (a.dim <= 32) forward<32>(g, st);
  else if (a.dim <= 64) forward<64>(g, st);
  else forward<128>(g, st);
}

void launch_train_attention_backward(const TrainAttention &a, float *delta, void *work, cudaStream_t st) {
  if (!a.bf16) return launch_train_attention_backward_f32(a, delta, work, st);
  const bool tc = train_attention_tc_supports(a, true);
  const long long tile = tc ? 128 : TA_B;  // the grids of all three kernels, before the first is launched
  for (const long long blocks : {(a.n + tile - 1) / tile * a.heads * a.streams, (a.m + tile - 1) / tile * a.groups * a.streams})
    if (blocks > 0x7fffffffLL) throw std::invalid_argument("attention: too many rows, heads and streams for one call");
  if (a.dim <= 64) launch_delta<8>(a, delta, st);
  else launch_delta<16>(a, delta, st);
  if (tc) return launch_train_attention_backward_tc(a, delta, st);
  if (a.dim <= 32) backward<32>(a, delta, st);
  else if (a.dim <= 64) backward<64>(a, delta, st);
  else backward<128>(a, delta, st);
}

}  // namespace lb

// Orthogonalised momentum of small matrices (smaller side up to 64): the whole step of a matrix in one launch, in 32 bits, by a
// thread-block cluster that keeps it in shared memory. The mathematics is that of orthogonal.cu.
//
// The larger side is cut over the C CTAs of the cluster; each holds 64 rows (the smaller side, zeros behind it) of its columns. A
// step of the iteration:
//   partial A = X_c X_c^T in every CTA; each sums 64 / C rows of A over the cluster in rank order and stores them in all CTAs
//   64 / C rows of B = b A + c A A, stored in all CTAs
//   X_c <- a X_c + B X_c, 64 columns at a time
// with a cluster barrier behind each. Norms are summed in 64 bits in rank order. 256 threads with 4 x 4 results each.
// Bound: latency, the barriers and the products of one CTA in turn (2 matrices of 64 x 256, five steps: 46 us a call,
// 129 as separate kernels).
#include "train_ops.cuh"
#include "gemm_tc.cuh"
#include "tc_ptx.cuh"

namespace lb {

namespace {

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f, NS_EPS = 1e-7f;
constexpr int SM_P = 64, SM_LD = SM_P + 4, SM_THREADS = 256, SM_MAX_COLS = 512;

constexpr int small_smem(int ldx) { return (SM_P * ldx + 3 * SM_P * SM_LD) * 4; }
static_assert(small_smem(SM_MAX_COLS + 4) <= 227 * 1024, "");

struct SmallArgs {
  MuonStep g;
  int p, q, cols, ldx;  // smaller and larger side, columns of a CTA, floats between rows of X
  int tall, ctas;
  float keep, rate;
};

__device__ __forceinline__ float *at(const MatView &v, long long off, long long r, long long c) {
  return reinterpret_cast<float *>(v.data + off + r * v.rs + c * v.cs);
}

// s[i][j] += rows (ty + 16 i) of a . rows (tx + 16 j) of b over k (a multiple of 4)
__device__ __forceinline__ void dot_tile(const float *a, int lda, const float *b, int ldb, int k, float (&s)[4][4]) {
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll 2
  for (int c = 0; c < k; c += 4) {
    float4 x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4 *>(a + (ty + 16 * i) * lda + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4 *>(b + (tx + 16 * j) * ldb + c);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        s[i][j] = fmaf(x[i].w, y[j].w, fmaf(x[i].z, y[j].z, fmaf(x[i].y, y[j].y, fmaf(x[i].x, y[j].x, s[i][j]))));
  }
}

__global__ void __launch_bounds__(SM_THREADS) muon_small_kernel(const __grid_constant__ SmallArgs s) {
  extern __shared__ float sm[];
  float *X = sm, *P = X + SM_P * s.ldx, *A = P + SM_P * SM_LD, *B = A + SM_P * SM_LD;
  __shared__ double red[8], part;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, lane = tid & 31;
  const int C = s.ctas, rank = (int)blockIdx.x % C;
  const long long batch = blockIdx.x / C;
  const MuonStep &g = s.g;
  const long long go = batch_offset(g.grads, batch), mo = g.step ? batch_offset(g.momentum, batch) : 0,
                  po = batch_offset(g.params, batch);
  const int first = rank * s.cols, mine = max(0, min(s.cols, s.q - first));
  pdl_launch_dependents();
  for (int e = tid; e < SM_P * s.ldx; e += SM_THREADS) X[e] = 0.f;
  __syncthreads();
  pdl_wait();
  // place e of this CTA's share: row i of the smaller side, column j of the larger
  auto place = [&](int e, int &i, int &j) {
    if (s.tall) {
      j = e / s.p;
      i = e - j * s.p;
    } else {
      i = e / mine;
      j = e - i * mine;
    }
  };
  double sum = 0.0;
  for (int e = tid; e < s.p * mine; e += SM_THREADS) {
    int i, j;
    place(e, i, j);
    const long long r = s.tall ? first + j : i, c = s.tall ? i : first + j;
    float u = *at(g.grads, go, r, c);
    if (g.step) {
      float *mom = at(g.momentum, mo, r, c);
      const float m = fmaf(g.mu, *mom, u);
      *mom = m;
      u = g.nesterov ? fmaf(g.mu, m, u) : m;
    }
    X[i * s.ldx + j] = u;
    sum += (double)u * (double)u;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) red[tid >> 5] = sum;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < SM_THREADS / 32; ++i) sum += red[i];
    part = sum;
  }
  __syncthreads();
  cluster_sync_all();
  sum = 0.0;
  for (int r = 0; r < C; ++r) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(cluster_map(smem_u32(&part), (unsigned)r)) : "memory");
    sum += v;
  }
  const double inv = 1.0 / (sqrt(sum) + (double)NS_EPS);
  for (int e = tid; e < s.p * mine; e += SM_THREADS) {
    int i, j;
    place(e, i, j);
    X[i * s.ldx + j] = (float)((double)X[i * s.ldx + j] * inv);
  }
  __syncthreads();
  const int k_cols = (mine + 3) & ~3, rows = SM_P / C, r0 = rank * rows;
  for (int step = 0; step < g.steps; ++step) {
    float acc[4][4] = {};
    dot_tile(X, s.ldx, X, s.ldx, k_cols, acc);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) P[(ty + 16 * i) * SM_LD + tx + 16 * j] = acc[i][j];
    __syncthreads();
    cluster_sync_all();
    for (int e = tid; e < rows * 16; e += SM_THREADS) {  // rows r0 .. r0 + rows - 1 of A, four columns at a time
      const unsigned off = (unsigned)((r0 + e / 16) * SM_LD + e % 16 * 4) * 4u, from = smem_u32(P) + off, to = smem_u32(A) + off;
      float4 v = ld_cluster_f4(cluster_map(from, 0u));
      for (int r = 1; r < C; ++r) {
        const float4 w = ld_cluster_f4(cluster_map(from, (unsigned)r));
        v = make_float4(v.x + w.x, v.y + w.y, v.z + w.z, v.w + w.w);
      }
      for (int r = 0; r < C; ++r) st_cluster_f4(cluster_map(to, (unsigned)r), v);
    }
    cluster_sync_all();
    for (int e = tid; e < rows * 16; e += SM_THREADS) {  // the same rows of B; A is symmetric: its row t for column t
      const int i = r0 + e / 16, j = e % 16 * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int t = 0; t < SM_P; ++t) {
        const float x = A[i * SM_LD + t];
        const float4 y = *reinterpret_cast<const float4 *>(A + t * SM_LD + j);
        v = make_float4(fmaf(x, y.x, v.x), fmaf(x, y.y, v.y), fmaf(x, y.z, v.z), fmaf(x, y.w, v.w));
      }
      const float4 a = *reinterpret_cast<const float4 *>(A + i * SM_LD + j);
      v = make_float4(fmaf(NS_B, a.x, NS_C * v.x), fmaf(NS_B, a.y, NS_C * v.y), fmaf(NS_B, a.z, NS_C * v.z), fmaf(NS_B, a.w, NS_C * v.w));
      const unsigned to = smem_u32(B) + (unsigned)(i * SM_LD + j) * 4u;
      for (int r = 0; r < C; ++r) st_cluster_f4(cluster_map(to, (unsigned)r), v);
    }
    cluster_sync_all();
    for (int c0 = 0; c0 < k_cols; c0 += 64) {  // rows ty + 16 i, columns c0 + 4 tx .. + 3
      const int c = c0 + 4 * tx;
      float4 v[4];
      if (c < k_cols) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int t = 0; t < SM_P; ++t) {
          const float4 y = *reinterpret_cast<const float4 *>(X + t * s.ldx + c);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = B[(ty + 16 * i) * SM_LD + t];
            v[i] = make_float4(fmaf(x, y.x, v[i].x), fmaf(x, y.y, v[i].y), fmaf(x, y.z, v[i].z), fmaf(x, y.w, v[i].w));
          }
        }
      }
      __syncthreads();
      if (c < k_cols) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float4 *x = reinterpret_cast<float4 *>(X + (ty + 16 * i) * s.ldx + c);
          const float4 o = *x;
          *x = make_float4(fmaf(NS_A, o.x, v[i].x), fmaf(NS_A, o.y, v[i].y), fmaf(NS_A, o.z, v[i].z), fmaf(NS_A, o.w, v[i].w));
        }
      }
    }
    __syncthreads();
  }
  for (int e = tid; e < s.p * mine; e += SM_THREADS) {
    int i, j;
    place(e, i, j);
    float *to = s.tall ? at(g.params, po, first + j, i) : at(g.params, po, i, first + j);
    const float v = X[i * s.ldx + j];
    *to = g.step ? fmaf(-s.rate, v, *to * s.keep) : v;
  }
  cluster_sync_all();  // no CTA's shared memory goes away while another reads it
}

}  // namespace

bool muon_small_supports(long long m, long long n) {
  const long long p = m < n ? m : n, q = m < n ? n : m;
  return p <= SM_P && q <= 8 * SM_MAX_COLS;
}

void launch_muon_small(const MuonStep &g, cudaStream_t st) {
  SmallArgs s{};
  const int m = (int)g.grads.rows, n = (int)g.grads.cols;
  s.g = g;
  s.tall = m > n;
  s.p = s.tall ? n : m;
  s.q = s.tall ? m : n;
  s.ctas = 1;
  while (s.ctas < 8 && s.q > 16 * s.ctas) s.ctas *= 2;
  s.cols = ((s.q + s.ctas - 1) / s.ctas + 3) & ~3;
  s.ldx = ((s.cols + 31) & ~31) + 4;
  s.keep = 1.f - g.lr * g.weight_decay;
  s.rate = g.lr * sqrtf(m > n ? (float)m / (float)n : 1.f);
  const size_t smem = small_smem(s.ldx);
  static SharedMemoryOnce once;  // the largest: the attribute is the kernel's, and calls of other threads want other sizes
  once.set(muon_small_kernel, small_smem(SM_MAX_COLS + 4));
  launch_pdl_cluster_x(muon_small_kernel, dim3((unsigned)(g.grads.batch * s.ctas)), dim3(SM_THREADS), smem, st, true,
                       (unsigned)s.ctas, s);
}

}  // namespace lb

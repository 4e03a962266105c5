// Orthogonalised momentum: the update of a weight matrix by the polynomial iteration
//   X = U / (|U| + 1e-7),  X <- a X + (b A + c A^2) X,  A = X X^T,  (a, b, c) = (3.4445, -4.7750, 2.0315)
// in the space of the matrix's smaller side, which drives its singular values towards 1; and the optimiser step with it,
//   momentum <- mu momentum + grad,  U = grad + mu momentum or momentum,
//   params <- (1 - lr decay) params - lr sqrt(max(1, m / n)) X.
// All matrices of a call have one shape and go through each step together. 32-bit products throughout.
#include "train_ops.cuh"

namespace lb {

namespace {

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f, NS_EPS = 1e-7f;
constexpr int NS_PARTS = 64;  // partial sums of a matrix's norm

struct NsWork {
  double *parts;      // [count][NS_PARTS]
  float *x, *y, *a, *b;
};

__device__ __forceinline__ float *element(const MatView &v, long long batch, long long r, long long c) {
  return reinterpret_cast<float *>(v.data + batch_offset(v, batch) + r * v.rs + c * v.cs);
}

// Momentum and the matrix to orthogonalise (in the orientation of x, whose rows are the smaller side), with partial sums of squares.
__global__ void __launch_bounds__(256) muon_begin_kernel(const __grid_constant__ MuonStep g, NsWork w, int tall) {
  const long long m = g.grads.rows, n = g.grads.cols, each = m * n, batch = blockIdx.y;
  double sum = 0.0;
  for (long long e = blockIdx.x * 256LL + threadIdx.x; e < each; e += 256LL * gridDim.x) {
    const long long r = e / n, c = e - r * n;
    const float grad = *element(g.grads, batch, r, c);
    float u = grad;
    if (g.step) {
      float *mom = element(g.momentum, batch, r, c);
      const float v = fmaf(g.mu, *mom, grad);
      *mom = v;
      u = g.nesterov ? fmaf(g.mu, v, grad) : v;
    }
    w.x[batch * each + (tall ? c * m + r : e)] = u;
    sum += (double)u * (double)u;
  }
  __shared__ double red[8];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) sum += red[i];
    w.parts[batch * NS_PARTS + blockIdx.x] = sum;
  }
}

__global__ void __launch_bounds__(256) muon_scale_kernel(NsWork w, long long each) {
  const long long batch = blockIdx.y;
  double sum = 0.0;
  for (int i = 0; i < (int)gridDim.x; ++i) sum += w.parts[batch * NS_PARTS + i];
  const float norm = (float)sqrt(sum) + NS_EPS;
  for (long long e = blockIdx.x * 256LL + threadIdx.x; e < each; e += 256LL * gridDim.x) w.x[batch * each + e] /= norm;
}

// y = p x + q y
__global__ void __launch_bounds__(256) muon_combine_kernel(float p, const float *x, float q, float *y, long long n) {
  for (long long e = blockIdx.x * 256LL + threadIdx.x; e < n; e += 256LL * gridDim.x) y[e] = fmaf(q, y[e], p * x[e]);
}

__global__ void __launch_bounds__(256) muon_end_kernel(const __grid_constant__ MuonStep g, const float *x, int tall, float keep,
                                                       float rate) {
  const long long m = g.grads.rows, n = g.grads.cols, each = m * n, batch = blockIdx.y;
  for (long long e = blockIdx.x * 256LL + threadIdx.x; e < each; e += 256LL * gridDim.x) {
    const long long r = e / n, c = e - r * n;
    const float v = x[batch * each + (tall ? c * m + r : e)];
    float *p = element(g.params, batch, r, c);
    *p = g.step ? fmaf(-rate, v, *p * keep) : v;
  }
}

MatView dense(float *p, long long count, long long rows, long long cols) {
  MatView v{};
  v.data = reinterpret_cast<char *>(p);
  v.nb = count > 1 ? 1 : 0;
  v.bd[0] = count;
  v.bs[0] = rows * cols * 4;
  v.batch = count;
  v.rows = rows;
  v.cols = cols;
  v.rs = cols * 4;
  v.cs = 4;
  return v;
}

MatView turned(MatView v) {
  std::swap(v.rows, v.cols);
  std::swap(v.rs, v.cs);
  return v;
}

unsigned blocks(long long n) { return (unsigned)((n + 255) / 256 < 148 * 8 ? (n + 255) / 256 : 148 * 8); }

}  // namespace

size_t muon_workspace_bytes(long long count, long long m, long long n) {
  const long long p = m < n ? m : n;
  return 256 + (size_t)count * (NS_PARTS * 8 + 2 * (size_t)m * n * 4 + 2 * (size_t)p * p * 4);
}

void launch_muon(const MuonStep &g, void *workspace, cudaStream_t st) {
  const long long m = g.grads.rows, n = g.grads.cols, count = g.grads.batch, each = m * n;
  const int tall = m > n;
  const long long p = tall ? n : m, q = tall ? m : n;
  NsWork w{};
  w.parts = static_cast<double *>(workspace);
  w.x = reinterpret_cast<float *>(w.parts + count * NS_PARTS);
  w.y = w.x + count * each;
  w.a = w.y + count * each;
  w.b = w.a + count * p * p;
  const dim3 grid((unsigned)((each + 255) / 256 < NS_PARTS ? (each + 255) / 256 : NS_PARTS), (unsigned)count);
  muon_begin_kernel<<<grid, 256, 0, st>>>(g, w, tall);
  LB_LAUNCH_CHECK();
  muon_scale_kernel<<<grid, 256, 0, st>>>(w, each);
  LB_LAUNCH_CHECK();
  for (int i = 0; i < g.steps; ++i) {
    const MatView x = dense(w.x, count, p, q), a = dense(w.a, count, p, p), b = dense(w.b, count, p, p);
    launch_gemm_simt(x, turned(x), a, p, p, q, GemmEpilogue{}, st);
    launch_gemm_simt(a, a, b, p, p, p, GemmEpilogue{}, st);
    muon_combine_kernel<<<blocks(count * p * p), 256, 0, st>>>(NS_B, w.a, NS_C, w.b, count * p * p);
    LB_LAUNCH_CHECK();
    launch_gemm_simt(b, x, dense(w.y, count, p, q), p, q, p, GemmEpilogue{}, st);
    muon_combine_kernel<<<blocks(count * each), 256, 0, st>>>(NS_A, w.x, 1.f, w.y, count * each);
    LB_LAUNCH_CHECK();
    std::swap(w.x, w.y);
  }
  const float rate = g.lr * sqrtf(m > n ? (float)m / (float)n : 1.f);
  muon_end_kernel<<<grid, 256, 0, st>>>(g, w.x, tall, 1.f - g.lr * g.weight_decay, rate);
  LB_LAUNCH_CHECK();
}

}  // namespace lb

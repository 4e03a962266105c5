// Clipped policy loss with a KL term, and its gradient in the logits:
//   logp_t = z_t[y_t] - log sum_c exp z_t[c],  z = logits / temp,  r = exp(logp - old)
//   loss   = sum_t w_t (-min(r A, clip(r, 1 - low, 1 + high) A) + beta (exp(d) - d - 1)) / sum_t w_t,  d = ref - logp
//   dlogits_t[c] = g_t (1[c = y_t] - exp(z_t[c] - lse_t)) / temp,
//   g_t = w_t / sum w (-[r A taken] r A + beta (1 - exp d))
// Rows of weight 0 are not read: their logp and gradient are 0. A target outside the vocabulary makes its row's logp and
// gradient, and the loss, NaN.
//
// One block per row: maximum and sum in one pass (a running pair per thread), the gradient in a second one. Row losses are
// summed in row order in 64 bits, so the loss does not depend on the order in which blocks finish.
// Bound: HBM, one read of the logits and one write of the gradient.
#include "train_ops.cuh"

#include <cuda_bf16.h>

namespace lb {

namespace {

typedef __nv_bfloat16 bf16;

constexpr int PL_THREADS = 256;
constexpr float PL_LOG2E = 1.4426950408889634f;

struct PlWork {
  double *row_loss;   // [rows]
  double *total;      // sum of the weights
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_float(float *p, float x) { *p = x; }
__device__ __forceinline__ void from_float(bf16 *p, float x) { *p = __float2bfloat16_rn(x); }

// Sum of `n` values in a fixed order by one block: thread sums over strides, then the threads in order of a tree.
template <typename T>
__device__ __forceinline__ double ordered_block_sum(const T *x, int n) {
  __shared__ double part[32];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) s += (double)x[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.0;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) s += part[i];
  return s;
}

__global__ void __launch_bounds__(1024) policy_weight_kernel(const float *weight, int rows, PlWork w) {
  const double s = ordered_block_sum(weight, rows);
  if (threadIdx.x == 0) *w.total = s;
}
__global__ void __launch_bounds__(1024) policy_join_kernel(int rows, PlWork w, float *loss) {
  const double s = ordered_block_sum(w.row_loss, rows);
  if (threadIdx.x == 0) *loss = (float)s;
}

// The row's share of the loss and its derivative in logp.
__device__ __forceinline__ void row_terms(const PolicyLoss &a, float logp, int row, float share, double &loss, float &g) {
  const float adv = a.advantage[row], r = expf(logp - a.old_logp[row]);
  const float low = 1.f - a.clip_low, high = 1.f + a.clip_high;
  const float taken = r * adv, clipped = fminf(fmaxf(r, low), high) * adv;
  float value = taken != taken ? taken : -fminf(taken, clipped);
  float d = (adv >= 0.f ? r <= high : r >= low) ? -taken : 0.f;
  if (r != r) d = r;
  if (a.kl_weight != 0.f) {
    const float diff = a.ref_logp[row] - logp, e = expf(diff);
    value += a.kl_weight * (fabsf(diff) < 0.25f ? expm1f(diff) - diff : e - diff - 1.f);
    d += a.kl_weight * -expm1f(diff);
  }
  loss = (double)value * (double)share;
  g = d * share;
}

template <typename T, int V>
struct Vec;
template <>
struct Vec<float, 4> { typedef float4 type; };
template <>
struct Vec<bf16, 8> { typedef uint4 type; };

template <typename T, int V>
__device__ __forceinline__ void unpack(const typename Vec<T, V>::type &u, float (&x)[V]) {
  const T *t = reinterpret_cast<const T *>(&u);
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = to_float(t[i]);
}

template <typename T, int V>  // V elements of 16 bytes at a time where rows allow it, else one at a time
__global__ void __launch_bounds__(PL_THREADS)
policy_rows_kernel(const __grid_constant__ PolicyLoss a, PlWork w, int vec, int dvec) {
  const int row = blockIdx.x, tid = threadIdx.x;
  const float weight = a.weight ? a.weight[row] : 1.f;
  const T *x = reinterpret_cast<const T *>(a.logits) + row * a.ld;
  T *dx = reinterpret_cast<T *>(a.dlogits) + row * a.dld;
  float share, slope, logp;
  const double total = a.weight ? *w.total : (double)a.rows;
  const int target = weight != 0.f ? a.targets[row] : 0;
  if (weight == 0.f || target < 0 || target >= a.vocab) {
    const float fill = weight == 0.f ? 0.f : NAN;
    if (tid == 0) {
      a.logp[row] = fill;
      w.row_loss[row] = fill;
    }
    if (a.dlogits)
      for (int c = tid; c < a.vocab; c += PL_THREADS) from_float(dx + c, fill);
    return;
  }
  share = (float)((double)weight / total);
  // exp2(z * f - top), top = max * f
  const float f = a.inv_temp * PL_LOG2E;
  float m = -INFINITY, s = 0.f;
  auto add = [&](float z) {
    if (z > m) {
      s = s * exp2f((m - z) * f);
      m = z;
    }
    s += z == -INFINITY ? 0.f : exp2f((z - m) * f);
  };
  if (vec) {
    const int n = a.vocab / V * V;
    for (int c = tid * V; c < n; c += PL_THREADS * V) {
      float z[V];
      unpack<T, V>(*reinterpret_cast<const typename Vec<T, V>::type *>(x + c), z);
      float top = z[0];
#pragma unroll
      for (int i = 1; i < V; ++i) top = fmaxf(top, z[i]);
      if (top > m) {
        s = s * exp2f((m - top) * f);
        m = top;
      }
      if (m != -INFINITY) {
#pragma unroll
        for (int i = 0; i < V; ++i) s += exp2f((z[i] - m) * f);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) s += z[i] == z[i] ? 0.f : z[i];
      }
    }
    for (int c = n + tid; c < a.vocab; c += PL_THREADS) add(to_float(x[c]));
  } else {
    for (int c = tid; c < a.vocab; c += PL_THREADS) add(to_float(x[c]));
  }
  __shared__ float sm_m[PL_THREADS / 32], sm_s[PL_THREADS / 32];
  auto join = [&](float m2, float s2) {
    const float top = fmaxf(m, m2);
    const float base = top == -INFINITY ? 0.f : top;
    s = s * exp2f((m - base) * f) + s2 * exp2f((m2 - base) * f);
    m = top;
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) join(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
  if ((tid & 31) == 0) {
    sm_m[tid >> 5] = m;
    sm_s[tid >> 5] = s;
  }
  __shared__ float out[2];
  __syncthreads();
  if (tid < 32) {
    m = tid < PL_THREADS / 32 ? sm_m[tid] : -INFINITY;
    s = tid < PL_THREADS / 32 ? sm_s[tid] : 0.f;
#pragma unroll
    for (int o = PL_THREADS / 64; o > 0; o >>= 1) join(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
    if (tid == 0) {
      logp = (to_float(x[target]) - m) * a.inv_temp - logf(s);
      double loss;
      row_terms(a, logp, row, share, loss, slope);
      a.logp[row] = logp;
      w.row_loss[row] = loss;
      out[0] = slope;
      out[1] = m;
      sm_s[0] = s;
    }
  }
  __syncthreads();
  if (!a.dlogits) return;
  slope = out[0] * a.inv_temp;
  m = out[1];
  const float per = -slope / sm_s[0];
  // the block's maximum subtracted before the factor: exact where the logits are near it
  if (vec && dvec) {
    const int n = a.vocab / V * V;
    for (int c = tid * V; c < n; c += PL_THREADS * V) {
      typename Vec<T, V>::type u = *reinterpret_cast<const typename Vec<T, V>::type *>(x + c);
      float z[V];
      unpack<T, V>(u, z);
      T *t = reinterpret_cast<T *>(&u);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float d = exp2f((z[i] - m) * f) * per;
        if (c + i == target) d += slope;
        from_float(t + i, d);
      }
      *reinterpret_cast<typename Vec<T, V>::type *>(dx + c) = u;
    }
    for (int c = n + tid; c < a.vocab; c += PL_THREADS) {
      float d = exp2f((to_float(x[c]) - m) * f) * per;
      if (c == target) d += slope;
      from_float(dx + c, d);
    }
  } else {
    for (int c = tid; c < a.vocab; c += PL_THREADS) {
      float d = exp2f((to_float(x[c]) - m) * f) * per;
      if (c == target) d += slope;
      from_float(dx + c, d);
    }
  }
}

template <typename T, int V>
void launch_rows(const PolicyLoss &a, const PlWork &w, cudaStream_t st) {
  const bool vec = a.ld % V == 0 && (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0;
  const bool dvec = a.dld % V == 0 && (reinterpret_cast<uintptr_t>(a.dlogits) & 15) == 0;
  policy_rows_kernel<T, V><<<(unsigned)a.rows, PL_THREADS, 0, st>>>(a, w, vec, dvec);
  LB_LAUNCH_CHECK();
}

}  // namespace

size_t policy_loss_workspace_bytes(long long rows) { return 256 + 8 * (size_t)rows; }

void launch_policy_loss(const PolicyLoss &a, void *workspace, cudaStream_t st) {
  PlWork w{reinterpret_cast<double *>(static_cast<char *>(workspace) + 256), static_cast<double *>(workspace)};
  if (a.weight) {
    policy_weight_kernel<<<1, 1024, 0, st>>>(a.weight, a.rows, w);
    LB_LAUNCH_CHECK();
  }
  if (a.bf16) launch_rows<bf16, 8>(a, w, st);
  else launch_rows<float, 4>(a, w, st);
  policy_join_kernel<<<1, 1024, 0, st>>>(a.rows, w, a.loss);
  LB_LAUNCH_CHECK();
}

}  // namespace lb

// Clipped policy loss with a KL term, and its gradient in the logits:
//   logp_t = z_t[y_t] - log sum_c exp z_t[c],  z = logits / temp,  r = exp(logp - old)
//   loss   = sum_t w_t (-min(r A, clip(r, 1 - low, 1 + high) A) + beta (exp(d) - d - 1)) / sum_t w_t,  d = ref - logp
//   dlogits_t[c] = g_t (1[c = y_t] - exp(z_t[c] - lse_t)) / temp,
//   g_t = w_t / sum w (-[r A taken] r A + beta (1 - exp d))
// Rows of weight 0 are not read: their logp and gradient are 0. A target outside the vocabulary makes its row's logp and
// gradient, and the loss, NaN.
//
// Up to 32768 columns a row stays in registers between its statistics and its gradient: read once, one exponential an element,
// written once. A warp takes a row of up to 1024 columns, 128, 256 or 512 threads with 64 elements each take longer ones. Beyond,
// 512 threads read the row twice, the second time from L2 (two blocks an SM, so that their rows fit there). Row losses are summed in
// row order in 64 bits, so the loss does not depend on the order in which blocks finish.
// Bound: HBM, one read of the logits and one write of the gradient. 4096 x 32000 in 32 bits, three in ten rows masked: 151 us for the rows'
// kernel (6.1 TB/s), 8 us around it; 4093 x 32000 in bfloat16: 89 us. All rows, whole calls, 32 bits and bfloat16: 4096 x 32000 175 and 102
// us (without the gradient 110 and 71); rows off 16-byte boundaries, element by element: 4096 x 16001 102 and 152, 4096 x 32001 248
// and 337; more than 32768 columns: 2048 x 64000 219 and 117, off boundaries 457 and 301.
// Exponentials are ex2.approx.ftz, good to 2^-22.
#include "train_ops.cuh"
#include "gemm_tc.cuh"
#include "tc_ptx.cuh"

#include <cuda_bf16.h>

namespace lb {

namespace {

typedef __nv_bfloat16 bf16;

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
  pdl_launch_dependents();
  const double s = ordered_block_sum(weight, rows);
  if (threadIdx.x == 0) *w.total = s;
}
__global__ void __launch_bounds__(1024) policy_join_kernel(int rows, PlWork w, float *loss) {
  pdl_wait();
  const double s = ordered_block_sum(w.row_loss, rows);
  if (threadIdx.x == 0) *loss = (float)s;
}

// 2^x; below 2^-126 0
__device__ __forceinline__ float pl_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What the loss of a row needs beside its logits; read before them, by the thread that finishes the row.
struct PlTerms {
  float adv, old, ref;
};
__device__ __forceinline__ PlTerms terms_of(const PolicyLoss &a, int row) {
  return PlTerms{a.advantage[row], a.old_logp[row], a.kl_weight != 0.f ? a.ref_logp[row] : 0.f};
}

// The row's share of the loss and its derivative in logp.
__device__ __forceinline__ void row_terms(const PolicyLoss &a, const PlTerms &t, float logp, float share, double &loss, float &g) {
  const float r = expf(logp - t.old);
  const float low = 1.f - a.clip_low, high = 1.f + a.clip_high;
  const float taken = r * t.adv, clipped = fminf(fmaxf(r, low), high) * t.adv;
  float value = taken != taken ? taken : -fminf(taken, clipped);
  float d = (t.adv >= 0.f ? r <= high : r >= low) ? -taken : 0.f;
  if (r != r) d = r;
  if (a.kl_weight != 0.f) {
    const float diff = t.ref - logp, e = expf(diff);
    value += a.kl_weight * (fabsf(diff) < 0.25f ? expm1f(diff) - diff : e - diff - 1.f);
    d += a.kl_weight * -expm1f(diff);
  }
  loss = (double)value * (double)share;
  g = d * share;
}

template <typename T>
struct PlVec;
template <>
struct PlVec<float> { static constexpr int V = 4; };
template <>
struct PlVec<bf16> { static constexpr int V = 8; };

// V consecutive elements; of those before `count`.
template <typename T>
__device__ __forceinline__ void load_vec(const T *p, float *x) {
  const uint4 u = __ldcs(reinterpret_cast<const uint4 *>(p));
  const T *t = reinterpret_cast<const T *>(&u);
#pragma unroll
  for (int i = 0; i < PlVec<T>::V; ++i) x[i] = to_float(t[i]);
}
__device__ __forceinline__ void store_vec(float *p, const float *x) {
  __stcs(reinterpret_cast<float4 *>(p), make_float4(x[0], x[1], x[2], x[3]));
}
__device__ __forceinline__ void store_vec(bf16 *p, const float *x) {  // (two to a conversion: one at a time a row's stores took twice as long)
  unsigned u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    u[i] = *reinterpret_cast<const unsigned *>(&v);
  }
  __stcs(reinterpret_cast<uint4 *>(p), make_uint4(u[0], u[1], u[2], u[3]));
}

struct PlForms {
  int vec, dvec;  // rows of logits and of the gradient on 16-byte boundaries
};

// What a row is: its share of the loss, or why it has none (fill: 0 for weight 0, NaN for a bad target).
struct PlRow {
  float weight;
  int target;
  bool fills;
  float fill;
};
__device__ __forceinline__ PlRow row_of(const PolicyLoss &a, int row) {
  PlRow r;
  r.weight = a.weight ? a.weight[row] : 1.f;
  r.target = r.weight != 0.f ? a.targets[row] : 0;
  r.fills = r.weight == 0.f || r.target < 0 || r.target >= a.vocab;
  r.fill = r.weight == 0.f ? 0.f : NAN;
  return r;
}
template <typename T>
__device__ __forceinline__ void fill_row(const PolicyLoss &a, const PlWork &w, const PlForms &f, int row, float fill, int at, int threads) {
  if (at == 0) {
    a.logp[row] = fill;
    w.row_loss[row] = fill;
  }
  if (!a.dlogits) return;
  constexpr int V = PlVec<T>::V;
  T *dx = reinterpret_cast<T *>(a.dlogits) + row * a.dld;
  int c = 0;
  if (f.dvec) {
    float x[V];
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = fill;
    for (c = at * V; c + V <= a.vocab; c += threads * V) store_vec(dx + c, x);
    c = a.vocab / V * V;
  }
  for (c += at; c < a.vocab; c += threads) from_float(dx + c, fill);
}
// 1 / the weights' sum, once it is there; 0 for weights without one, all zero or not.
__device__ __forceinline__ double inverse_total(const PolicyLoss &a, const PlWork &w) {
  const double total = a.weight ? *static_cast<volatile double *>(w.total) : (double)a.rows;
  return total == 0.0 ? 0.0 : 1.0 / total;
}
// Loss and slope of a row from its statistics, by one thread: the slope in the logits comes back.
__device__ __forceinline__ float finish_row(const PolicyLoss &a, const PlWork &w, int row, const PlTerms &t, float share, float z, float top,
                                            float sum) {
  const float logp = (z - top) * a.inv_temp - logf(sum);
  double loss;
  float slope;
  row_terms(a, t, logp, share, loss, slope);
  a.logp[row] = logp;
  w.row_loss[row] = loss;
  return slope * a.inv_temp;
}

// THREADS to a row, ROWS rows to a block (THREADS = 32: a warp each), up to 64 (32) elements to a thread, all in registers.
template <typename T, int THREADS, int ROWS>
__global__ void __launch_bounds__(THREADS *ROWS)
policy_row_kernel(const __grid_constant__ PolicyLoss a, PlWork w, PlForms f) {
  constexpr int V = PlVec<T>::V, N = (THREADS == 32 ? 32 : 64) / V, WARPS = THREADS / 32;
  const int at = threadIdx.x % THREADS, row = blockIdx.x * ROWS + threadIdx.x / THREADS;
  __shared__ float red[2][WARPS];
  __shared__ float out[1];
  if (ROWS > 1 && row >= a.rows) return;  // (a whole warp)
  const PlRow r = row_of(a, row);
  if (r.fills) {
    if (a.weight) pdl_wait();  // (an earlier call's sums have been read)
    return fill_row<T>(a, w, f, row, r.fill, at, THREADS);
  }
  const T *x = reinterpret_cast<const T *>(a.logits) + row * a.ld;
  T *dx = reinterpret_cast<T *>(a.dlogits) + row * a.dld;
  const PlTerms t = at == 0 ? terms_of(a, row) : PlTerms{};
  const float zt = at == 0 ? to_float(x[r.target]) : 0.f;
  float z[N * V];
  // vectors: element (i THREADS + at) V + j; one at a time: (i V + j) THREADS + at
  auto place = [&](int i, int j) { return f.vec ? (i * THREADS + at) * V + j : (i * V + j) * THREADS + at; };
  if (f.vec) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * THREADS + at) * V;
      if (c + V <= a.vocab) {
        load_vec(x + c, z + i * V);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) z[i * V + j] = c + j < a.vocab ? to_float(x[c + j]) : -INFINITY;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N * V; ++i) z[i] = i * THREADS + at < a.vocab ? to_float(x[i * THREADS + at]) : -INFINITY;
  }
  auto all = [&](float v, bool sum, int which) {  // over the row's threads
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float u = __shfl_xor_sync(0xffffffffu, v, o);
      v = sum ? v + u : fmaxf(v, u);
    }
    if (WARPS == 1) return v;
    if ((at & 31) == 0) red[which][at >> 5] = v;
    __syncthreads();
    v = red[which][0];
#pragma unroll
    for (int i = 1; i < WARPS; ++i) v = sum ? v + red[which][i] : fmaxf(v, red[which][i]);
    return v;
  };
  float top = z[0];
#pragma unroll
  for (int i = 1; i < N * V; ++i) top = fmaxf(top, z[i]);
  top = all(top, false, 0);
  const float factor = a.inv_temp * PL_LOG2E;
  float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N * V; ++i) {
    z[i] = pl_exp2((z[i] - top) * factor);
    s4[i & 3] += z[i];
  }
  const float sum = all((s4[0] + s4[1]) + (s4[2] + s4[3]), true, 1);
  if (a.weight) pdl_wait();  // the weights' sum is there
  float slope;
  const float share = at == 0 ? (float)((double)r.weight * inverse_total(a, w)) : 0.f;
  if (WARPS == 1) {
    slope = at == 0 ? finish_row(a, w, row, t, share, zt, top, sum) : 0.f;
    slope = __shfl_sync(0xffffffffu, slope, 0);
  } else {
    if (at == 0) out[0] = finish_row(a, w, row, t, share, zt, top, sum);
    __syncthreads();
    slope = out[0];
  }
  if (!a.dlogits) return;
  const float per = -slope / sum;
#pragma unroll
  for (int i = 0; i < N * V; ++i) z[i] *= per;
  if (f.vec && f.dvec) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * THREADS + at) * V;
      if (c <= r.target && r.target < c + V) {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (c + j == r.target) z[i * V + j] += slope;
      }
      if (c + V <= a.vocab) {
        store_vec(dx + c, z + i * V);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (c + j < a.vocab) from_float(dx + c + j, z[i * V + j]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = place(i, j);
        if (c < a.vocab) from_float(dx + c, c == r.target ? z[i * V + j] + slope : z[i * V + j]);
      }
  }
}

// The same for rows of 8193 to 32768 columns on 16-byte boundaries, by blocks that walk rows and bring the next one into shared memory while
// they work on one. 32 bits: a block of 1024 threads per SM, 32 exponentials to a thread in registers. bfloat16: two blocks of 512 per SM,
// whose phases overlap, with 64 elements to a thread as they are (32 registers; the exponentials are taken twice). 4093 x 32000 in bfloat16:
// 120 us the first way, 87 us the second.
template <typename T>
struct PlStream;
template <>
struct PlStream<float> { static constexpr int THREADS = 1024, BLOCKS = 1; };
template <>
struct PlStream<bf16> { static constexpr int THREADS = 512, BLOCKS = 2; };

__device__ __forceinline__ float2 two_of(unsigned u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

template <typename T>
__global__ void __launch_bounds__(PlStream<T>::THREADS, PlStream<T>::BLOCKS)
policy_stream_kernel(const __grid_constant__ PolicyLoss a, PlWork w, PlForms f) {
  constexpr int THREADS = PlStream<T>::THREADS, V = PlVec<T>::V, N = 32768 / THREADS / V, WARPS = THREADS / 32;
  constexpr bool HALF = sizeof(T) == 2;
  extern __shared__ __align__(16) unsigned char sm_row[];
  __shared__ __align__(8) unsigned long long bar_word;
  __shared__ float red[2][WARPS], out[2];
  __shared__ int abort_word;
  const int tid = threadIdx.x, whole = a.vocab / V * V;
  const unsigned bar = smem_u32(&bar_word);
  auto fetch = [&](int row, const PlRow &r) {  // by one thread: the row's whole vectors, if there is such a row and it is read at all
    if (row >= a.rows || r.fills) return;
    const unsigned bytes = (unsigned)whole * (unsigned)sizeof(T);
    mbar_expect_tx(bar, bytes);
    bulk_load(smem_u32(sm_row), reinterpret_cast<const T *>(a.logits) + row * a.ld, bytes, bar);
  };
  PlRow r = row_of(a, blockIdx.x);
  if (tid == 0) {
    mbar_init(bar, 1);
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    fetch(blockIdx.x, r);
  }
  __syncthreads();
  if (a.weight) pdl_wait();
  unsigned phase = 0;
  const float factor = a.inv_temp * PL_LOG2E;
  const double inverse = tid == 0 ? inverse_total(a, w) : 0.0;
  // A row that did not come in time: it and all after it are NaN (the barrier's phases say nothing any more, the shared memory may hold any
  // row), and the CTA stays until the copy has landed, within the limit.
  bool lost = false;
  PlRow next;
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x, r = next) {
    const int after = row + gridDim.x;
    next = row_of(a, after < a.rows ? after : row);
    if (r.fills) {
      if (tid == 0 && !lost) fetch(after, next);
      fill_row<T>(a, w, f, row, r.fill, tid, THREADS);
      continue;
    }
    if (lost) {
      fill_row<T>(a, w, f, row, NAN, tid, THREADS);
      continue;
    }
    const T *x = reinterpret_cast<const T *>(a.logits) + row * a.ld;
    T *dx = reinterpret_cast<T *>(a.dlogits) + row * a.dld;
    const PlTerms t = tid == 0 ? terms_of(a, row) : PlTerms{};
    const float zt = tid == 0 ? to_float(x[r.target]) : 0.f, share = (float)((double)r.weight * inverse);
    const int last = whole + tid;  // fewer than V columns behind the vectors, one to a thread
    float tail = last < a.vocab ? to_float(x[last]) : -INFINITY;
    const bool there = mbar_wait(bar, phase & 1u, reinterpret_cast<volatile int *>(&abort_word), nullptr, 141);
    ++phase;
    // 16 bytes each: four values or eight; 0xff80 is -infinity
    uint4 z[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * THREADS + tid) * V;
      const unsigned none = HALF ? 0xff80ff80u : 0xff800000u;
      z[i] = c < whole ? *reinterpret_cast<const uint4 *>(sm_row + (size_t)c * sizeof(T)) : make_uint4(none, none, none, none);
    }
    lost = !__syncthreads_and(there);
    if (lost) {
      fill_row<T>(a, w, f, row, NAN, tid, THREADS);
      continue;
    }
    if (tid == 0) fetch(after, next);
    auto all = [&](float v, bool sum, int which) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float u = __shfl_xor_sync(0xffffffffu, v, o);
        v = sum ? v + u : fmaxf(v, u);
      }
      if ((tid & 31) == 0) red[which][tid >> 5] = v;
      __syncthreads();
      v = red[which][tid % WARPS];
#pragma unroll
      for (int o = WARPS / 2; o > 0; o >>= 1) {
        const float u = __shfl_xor_sync(0xffffffffu, v, o);
        v = sum ? v + u : fmaxf(v, u);
      }
      return v;
    };
    float top;
    if (HALF) {
      __nv_bfloat162 m4[4];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const __nv_bfloat162 *e = reinterpret_cast<const __nv_bfloat162 *>(&z[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) m4[j] = i == 0 ? e[j] : __hmax2(m4[j], e[j]);
      }
      const float2 m = __bfloat1622float2(__hmax2(__hmax2(m4[0], m4[1]), __hmax2(m4[2], m4[3])));
      top = fmaxf(fmaxf(m.x, m.y), tail);
    } else {
      top = tail;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float4 e = *reinterpret_cast<const float4 *>(&z[i]);
        top = fmaxf(fmaxf(fmaxf(top, e.x), fmaxf(e.y, e.z)), e.w);
      }
    }
    top = all(top, false, 0);
    auto weight_of = [&](float v) { return pl_exp2((v - top) * factor); };
    tail = weight_of(tail);
    float s4[4] = {tail, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (HALF) {
        const unsigned u[4] = {z[i].x, z[i].y, z[i].z, z[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 v = two_of(u[j]);
          s4[j] += weight_of(v.x) + weight_of(v.y);
        }
      } else {
        float4 &e = *reinterpret_cast<float4 *>(&z[i]);
        e = make_float4(weight_of(e.x), weight_of(e.y), weight_of(e.z), weight_of(e.w));
        s4[0] += e.x;
        s4[1] += e.y;
        s4[2] += e.z;
        s4[3] += e.w;
      }
    }
    const float sum = all((s4[0] + s4[1]) + (s4[2] + s4[3]), true, 1);
    if (tid == 0) {
      out[0] = finish_row(a, w, row, t, share, zt, top, sum);
      out[1] = weight_of(zt);
    }
    __syncthreads();
    if (!a.dlogits) continue;
    const float slope = out[0], per = -slope / sum;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * THREADS + tid) * V;
      if (c >= whole) continue;
      float d[V];
      if (HALF) {
        const unsigned u[4] = {z[i].x, z[i].y, z[i].z, z[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 v = two_of(u[j]);
          d[(2 * j) % V] = weight_of(v.x) * per;
          d[(2 * j + 1) % V] = weight_of(v.y) * per;
        }
      } else {
        const float4 e = *reinterpret_cast<const float4 *>(&z[i]);
        d[0] = e.x * per;
        d[1] = e.y * per;
        d[2] = e.z * per;
        d[3] = e.w * per;
      }
      if (f.dvec) {
        store_vec(dx + c, d);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) from_float(dx + c + j, d[j]);
      }
    }
    if (last < a.vocab) from_float(dx + last, tail * per);
    // the target's own, behind what its thread has stored there
    if (r.target < whole ? tid == r.target / V % THREADS : last == r.target) from_float(dx + r.target, fmaf(out[1], per, slope));
  }
  if (lost && tid == 0) {
    const unsigned long long limit = global_timer() + WAIT_LIMIT_NS;
    while (!mbar_try_wait(bar, (phase - 1u) & 1u) && global_timer() < limit) {}
  }
}

// Any number of columns: a running maximum and sum per thread, then the row again.
constexpr int PL_LONG = 512;
template <typename T>
__global__ void __launch_bounds__(PL_LONG, 2)
policy_long_kernel(const __grid_constant__ PolicyLoss a, PlWork w, PlForms f) {
  constexpr int V = PlVec<T>::V, AHEAD = 4, WARPS = PL_LONG / 32;
  const int row = blockIdx.x, tid = threadIdx.x;
  const PlRow r = row_of(a, row);
  if (r.fills) {
    if (a.weight) pdl_wait();
    return fill_row<T>(a, w, f, row, r.fill, tid, PL_LONG);
  }
  const T *x = reinterpret_cast<const T *>(a.logits) + row * a.ld;
  T *dx = reinterpret_cast<T *>(a.dlogits) + row * a.dld;
  const float factor = a.inv_temp * PL_LOG2E;
  float m = -INFINITY, s = 0.f;
  auto add = [&](const float *z, int n) {
    float top = z[0];
    for (int i = 1; i < n; ++i) top = fmaxf(top, z[i]);
    if (top > m) {
      s *= pl_exp2((m - top) * factor);
      m = top;
    }
    const float base = m == -INFINITY ? 0.f : m;
    for (int i = 0; i < n; ++i) s += pl_exp2((z[i] - base) * factor);
  };
  const int whole = f.vec ? a.vocab / V * V : 0;  // columns that vectors cover
  for (int c = tid * V; c < whole; c += PL_LONG * V * AHEAD) {
    float z[AHEAD * V];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int at = c + u * PL_LONG * V;
      if (at < whole) {
        const uint4 q = *reinterpret_cast<const uint4 *>(x + at);
        const T *t = reinterpret_cast<const T *>(&q);
#pragma unroll
        for (int i = 0; i < V; ++i) z[u * V + i] = to_float(t[i]);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) z[u * V + i] = -INFINITY;
      }
    }
    add(z, AHEAD * V);
  }
  for (int c = whole + tid; c < a.vocab; c += PL_LONG) {
    const float z = to_float(x[c]);
    add(&z, 1);
  }
  __shared__ float sm_m[WARPS], sm_s[WARPS], out[3];
  auto join = [&](float m2, float s2) {
    const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.f : top;
    s = s * pl_exp2((m - base) * factor) + s2 * pl_exp2((m2 - base) * factor);
    m = top;
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    join(m2, s2);
  }
  if ((tid & 31) == 0) {
    sm_m[tid >> 5] = m;
    sm_s[tid >> 5] = s;
  }
  __syncthreads();
  if (tid < 32) {
    m = tid < WARPS ? sm_m[tid] : -INFINITY;
    s = tid < WARPS ? sm_s[tid] : 0.f;
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
      join(m2, s2);
    }
    if (tid == 0) {
      if (a.weight) pdl_wait();  // the weights' sum is there
      if (m == -INFINITY) s = NAN;  // a row that is masked altogether is not a distribution
      out[0] = finish_row(a, w, row, terms_of(a, row), (float)((double)r.weight * inverse_total(a, w)), to_float(x[r.target]), m, s);
      out[1] = m;
      out[2] = s;
    }
  }
  __syncthreads();
  if (!a.dlogits) return;
  const float slope = out[0], per = -slope / out[2];
  m = out[1];
  const int both = f.dvec ? whole : 0;
  for (int c = tid * V; c < both; c += PL_LONG * V * AHEAD) {
    uint4 q[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (c + u * PL_LONG * V < both) q[u] = __ldcs(reinterpret_cast<const uint4 *>(x + c + u * PL_LONG * V));
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int at = c + u * PL_LONG * V;
      if (at >= both) break;
      const T *t = reinterpret_cast<const T *>(&q[u]);
      float d[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        d[i] = pl_exp2((to_float(t[i]) - m) * factor) * per;
        if (at + i == r.target) d[i] += slope;
      }
      store_vec(dx + at, d);
    }
  }
  for (int c = both + tid; c < a.vocab; c += PL_LONG) {
    const float d = pl_exp2((to_float(x[c]) - m) * factor) * per;
    from_float(dx + c, c == r.target ? d + slope : d);
  }
}

template <typename T>
void launch_rows(const PolicyLoss &a, const PlWork &w, cudaStream_t st) {
  constexpr int V = PlVec<T>::V;
  PlForms f;
  f.vec = (a.rows == 1 || a.ld % V == 0) && (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0;
  f.dvec = (a.rows == 1 || a.dld % V == 0) && (reinterpret_cast<uintptr_t>(a.dlogits) & 15) == 0;
  const bool pdl = a.weight != nullptr;  // behind the sum of the weights, which was launched the ordinary way: what came before it is done
  const unsigned rows = (unsigned)a.rows;
  if (a.vocab <= 1024) launch_pdl(policy_row_kernel<T, 32, 4>, dim3((rows + 3) / 4), dim3(128), 0, st, pdl, a, w, f);
  else if (a.vocab <= 8192) launch_pdl(policy_row_kernel<T, 128, 1>, dim3(rows), dim3(128), 0, st, pdl, a, w, f);
  else if (f.vec && a.vocab <= 32768) {
    constexpr unsigned BLOCKS = 148 * PlStream<T>::BLOCKS;
    static SharedMemoryOnce once;
    once.set(policy_stream_kernel<T>, 32768 * (int)sizeof(T));
    launch_pdl(policy_stream_kernel<T>, dim3(rows < BLOCKS ? rows : BLOCKS), dim3(PlStream<T>::THREADS), (size_t)a.vocab * sizeof(T), st,
               pdl, a, w, f);
  } else if (a.vocab <= 16384) launch_pdl(policy_row_kernel<T, 256, 1>, dim3(rows), dim3(256), 0, st, pdl, a, w, f);
  else if (a.vocab <= 32768) launch_pdl(policy_row_kernel<T, 512, 1>, dim3(rows), dim3(512), 0, st, pdl, a, w, f);
  else launch_pdl(policy_long_kernel<T>, dim3(rows), dim3(PL_LONG), 0, st, pdl, a, w, f);
}

}  // namespace

size_t policy_loss_workspace_bytes(long long rows) { return 256 + 8 * (size_t)rows; }

void launch_policy_loss(const PolicyLoss &a, void *workspace, cudaStream_t st) {
  PlWork w{reinterpret_cast<double *>(static_cast<char *>(workspace) + 256), static_cast<double *>(workspace)};
  if (a.weight) {
    policy_weight_kernel<<<1, 1024, 0, st>>>(a.weight, a.rows, w);
    LB_LAUNCH_CHECK();
  }
  if (a.bf16) launch_rows<bf16>(a, w, st);
  else launch_rows<float>(a, w, st);
  launch_pdl(policy_join_kernel, dim3(1), dim3(1024), 0, st, true, a.rows, w, a.loss);
}

}  // namespace lb

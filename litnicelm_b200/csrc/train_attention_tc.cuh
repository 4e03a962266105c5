// What the tensor-core kernels of the training attention share (train_attention_tc.cu in bfloat16, train_attention_f32.cu in 32
// bits): arguments, which tile a CTA has, small helpers.
#pragma once

#include "train_ops.cuh"
#include "gemm_tc.cuh"
#include "tc_ptx.cuh"

#include <cuda_bf16.h>

namespace lb {

namespace {

typedef __nv_bfloat16 bf16;

constexpr int TT_B = 128;
constexpr int TT_SLAB = 128 * 128;  // 128 rows of 64 elements
constexpr float TT_NEG = -3.0e38f, TT_SLACK = 8.f, TT_LOG2E = 1.4426950408889634f;  // TT_NEG: below every score
constexpr float TT_FAR = 268435456.f;  // 2^28: half a step of a score there is 2^3 to 2^4, of an exponent

__device__ __forceinline__ float tt_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ unsigned tt_pack(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const unsigned *>(&v);
}

// Two 32-bit operations in one instruction.
__device__ __forceinline__ unsigned long long tt_two(float a, float b) {
  return (unsigned long long)__float_as_uint(a) | (unsigned long long)__float_as_uint(b) << 32;
}
__device__ __forceinline__ float tt_lo(unsigned long long x) { return __uint_as_float((unsigned)x); }
__device__ __forceinline__ float tt_hi(unsigned long long x) { return __uint_as_float((unsigned)(x >> 32)); }
__device__ __forceinline__ unsigned long long tt_fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ unsigned long long tt_add2(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ unsigned long long tt_mul2(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// The largest of three, NaN if one of them is.
__device__ __forceinline__ float tt_max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

struct TtArgs {
  int n, m, heads, groups, share, streams, dim, tiles;
  TrainSpan span;
  int seen;
  const int *lengths;
  float scale, factor;   // factor = scale * log2(e)
  float *lse;
  float *delta;
  HeadView o1, o2;       // out | dq | dk, dv
  HeadView q, k, v;      // of the bfloat16 forward kernels (tt_row_again)
  int vec;               // results' rows on 16-byte boundaries
};

struct TtPlace {
  int tile, head, stream, keys;
};
__device__ __forceinline__ TtPlace tt_place(const TtArgs &a, int heads, bool last_first, int ctas, int block) {  // ctas: to a tile
  const int each = heads * a.streams, b = block / ctas;
  const int t = b / each, rest = b - t * each;
  TtPlace p;
  p.tile = last_first ? a.tiles - 1 - t : t;
  p.stream = rest / heads;
  p.head = rest - p.stream * heads;
  p.keys = a.lengths ? max(0, min(a.seen, a.lengths[p.stream])) : a.seen;
  return p;
}
__device__ __forceinline__ TtPlace tt_place(const TtArgs &a, int heads, bool last_first, int ctas = 1) {
  return tt_place(a, heads, last_first, ctas, (int)blockIdx.x);
}

// A value that all lanes have, known as such to the compiler: what is computed from it stays in uniform registers.
__device__ __forceinline__ int tt_uniform(int x) { return __reduce_max_sync(0xffffffffu, x); }

// Blocks that have not started, taken over by running ones (cluster launch control): a block's warps go on with the next tile while
// its last results are on their way, nothing is set up again, and whoever is free first takes the next. Warp 0 asks, with the last
// loads of a block (sooner, and others would be free for it first), and passes the blocks that have work on to `readers` warps, in two
// places in turn; what a block without work leaves it does itself, so a reader that is one or two blocks ahead of the others
// never waits for them. 72 bytes of shared memory from `at` on.
struct TtNext {
  unsigned at;
  int asks = 0;
  __device__ __forceinline__ unsigned got() const { return at + 24u; }
  __device__ __forceinline__ unsigned full(int w) const { return at + 32u + 8u * (w & 1); }
  __device__ __forceinline__ unsigned empty(int w) const { return at + 48u + 8u * (w & 1); }
  __device__ __forceinline__ unsigned drained() const { return at + 64u; }  // of a CTA that gave up
  __device__ __forceinline__ void init(int readers) const {
    for (int w = 0; w < 2; ++w) {
      mbar_init(full(w), 1);
      mbar_init(empty(w), readers);
    }
    mbar_init(got(), 1);
    mbar_init(drained(), 1);
  }
  // These waits go on in a CTA that gave up on another: each block that it has taken gets its results, if only NaN.
  static __device__ __forceinline__ bool wait(unsigned bar, unsigned parity) {
    bool ok = true;
    if (!mbar_try_wait(bar, parity)) {
      const unsigned long long limit = global_timer() + 16 * WAIT_LIMIT_NS;
      while (ok && !mbar_try_wait(bar, parity)) ok = global_timer() < limit;
    }
    return __all_sync(0xffffffffu, ok);
  }
  // Not again after an answer of none.
  __device__ __forceinline__ void ask(int lane) const {
    if (lane == 0) {
      mbar_expect_tx(got(), 16u);
      asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(at), "r"(got())
                   : "memory");
    }
    __syncwarp();
  }
  // The block asked for, or -1.
  __device__ __forceinline__ int answer() {
    if (!wait(got(), (unsigned)asks++ & 1u)) return -1;
    unsigned some, block;
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t"
        "ld.shared.b128 r, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
        "selp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
        : "=r"(some), "=r"(block)
        : "r"(at)
        : "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    return tt_uniform(some ? (int)block : -1);
  }
  // The w-th block with work (or -1, the end) for the readers.
  __device__ __forceinline__ void push(int w, int block, int lane) const {
    if (!wait(empty(w), ((unsigned)(w >> 1) & 1u) ^ 1u)) return;
    if (lane == 0) {
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + 16u + 4u * (w & 1)), "r"(block) : "memory");
      mbar_arrive(full(w));
    }
    __syncwarp();
  }
  __device__ __forceinline__ int take(int w, int lane) const {
    if (!wait(full(w), (unsigned)(w >> 1) & 1u)) return -1;
    int block;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(block) : "r"(at + 16u + 4u * (w & 1)) : "memory");
    __syncwarp();
    if (lane == 0) mbar_arrive(empty(w));
    return tt_uniform(block);
  }
};

__device__ __forceinline__ void tt_alloc(volatile unsigned *holder, unsigned cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void *)holder)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}


TtArgs tt_args(const TrainAttention &a, int rows) {
  TtArgs t{};
  t.n = a.n;
  t.m = a.m;
  t.heads = a.heads;
  t.groups = a.groups;
  t.share = a.heads / a.groups;
  t.streams = a.streams;
  t.dim = a.dim;
  t.tiles = (rows + TT_B - 1) / TT_B;
  t.span = TrainSpan{a.first, a.window, a.causal};
  t.seen = a.seen;
  t.lengths = a.lengths;
  t.scale = a.scale;
  t.factor = a.scale * TT_LOG2E;
  t.lse = a.lse;
  return t;
}

unsigned tt_grid(const TtArgs &t, int heads, int ctas = 1) {
  const long long blocks = (long long)t.tiles * heads * t.streams * ctas;
  if (blocks > 0x7fffffffLL) throw std::invalid_argument("attention: too many rows, heads and streams for one call");
  return (unsigned)blocks;
}

}  // namespace

}  // namespace lb

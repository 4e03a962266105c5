// Operators of a training step on the caller's device memory (section 4 of the C header): attention whose backward pass
// recomputes the probabilities, the clipped policy loss, orthogonalised momentum. Launchers of the kernel files; the checks
// of arguments are in train_api.cu.
#pragma once

#include "common.cuh"

namespace lb {

// [streams, rows, heads, dim] with element strides.
struct HeadView {
  char *p = nullptr;
  long long s = 0, r = 0, h = 0, c = 0;
};

struct TrainAttention {
  HeadView q, k, v, out, dout, dq, dk, dv;
  float *lse = nullptr;            // [streams, heads, n]
  const int *lengths = nullptr;    // keys of each stream, device
  int streams = 0, n = 0, m = 0, heads = 0, groups = 0, dim = 0;
  float scale = 1.f;
  int causal = 0, first = 0, window = 0;
  int seen = 0;                    // keys from here on are behind every row, as those from a stream's length on
  int bf16 = 0;
};

// Key j is seen by row i (position first + i) if j < m, j < lengths, with causal j <= first + i, with a window
// j > first + i - window.
struct TrainSpan {
  int first, window, causal;
  __host__ __device__ int lo(int i) const { return window > 0 ? (first + i - window + 1 > 0 ? first + i - window + 1 : 0) : 0; }
  __host__ __device__ int end(int i, int keys) const { return causal && first + i + 1 < keys ? first + i + 1 : keys; }
  // Of n rows, those from here on see no key.
  __host__ __device__ int rows_end(int n, int keys) const {
    const long long past = keys <= 0 ? 0 : window > 0 ? (long long)keys - 1 + window - first : n;
    return past < 0 ? 0 : past < n ? (int)past : n;
  }
};

constexpr int TRAIN_MAX_DIM = 128;

// train_attention.cu: bfloat16 of any sizes and strides, 32-bit arithmetic throughout; dispatches to the two below. `work`:
// train_attention_f32_workspace bytes for 32-bit operands.
void launch_train_attention_forward(const TrainAttention &a, void *work, cudaStream_t st);
void launch_train_attention_backward(const TrainAttention &a, float *delta, void *work, cudaStream_t st);

// train_attention_tc.cu: bfloat16 on the tensor cores, where every operand can be addressed by TMA
bool train_attention_tc_supports(const TrainAttention &a, bool backward);
void launch_train_attention_forward_tc(const TrainAttention &a, cudaStream_t st);
void launch_train_attention_backward_tc(const TrainAttention &a, float *delta, cudaStream_t st);

// train_attention_f32.cu: 32 bits on the tensor cores
size_t train_attention_f32_workspace(long long streams, long long n, long long m, long long heads, long long groups, long long dim,
                                     bool backward);
void launch_train_attention_forward_f32(const TrainAttention &a, void *work, cudaStream_t st);
void launch_train_attention_backward_f32(const TrainAttention &a, float *delta, void *work, cudaStream_t st);

struct PolicyLoss {
  const char *logits = nullptr;
  char *dlogits = nullptr;         // null: no gradient; may be logits
  long long ld = 0, dld = 0;       // elements
  const int *targets = nullptr;
  const float *old_logp = nullptr, *advantage = nullptr, *ref_logp = nullptr, *weight = nullptr;
  float *loss = nullptr, *logp = nullptr;
  int rows = 0, vocab = 0, bf16 = 0;
  float inv_temp = 1.f, clip_low = 0.f, clip_high = 0.f, kl_weight = 0.f;
};
size_t policy_loss_workspace_bytes(long long rows);
void launch_policy_loss(const PolicyLoss &a, void *workspace, cudaStream_t st);

struct MuonStep {
  int step = 0;                    // 0: out = orthogonal factor of grads; 1: the optimiser step
  MatView grads, momentum, params; // params: the result where step is 0
  float lr = 0.f, mu = 0.f, weight_decay = 0.f;
  int nesterov = 0, steps = 5;
};
size_t muon_workspace_bytes(long long count, long long m, long long n);
void launch_muon(const MuonStep &a, void *workspace, cudaStream_t st);
// orthogonal_small.cu: small matrices in one launch
bool muon_small_supports(long long m, long long n);
void launch_muon_small(const MuonStep &a, cudaStream_t st);

}  // namespace lb

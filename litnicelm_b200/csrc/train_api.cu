// Entry points of the training operators on the caller's device memory: every argument is checked here, before anything is
// enqueued, and no exception leaves.
#include "train_ops.cuh"

#include <cmath>
#include <cstring>

using namespace lb;

namespace {

constexpr long long MAX_EXTENT = 1 << 30;

int refuse(int code, const std::string &text) {
  set_call_error(text.c_str());
  return code;
}

template <typename F>
int guarded(const char *who, F f) {
  try {
    f();
    return LITNICE_B200_OK;
  } catch (const std::invalid_argument &e) {
    return refuse(LITNICE_B200_EINVAL, std::string(who) + ": " + e.what());
  } catch (const std::exception &e) {
    return refuse(LITNICE_B200_ECUDA, std::string(who) + ": " + e.what());
  } catch (...) {
    return refuse(LITNICE_B200_ECUDA, std::string(who) + ": unknown error");
  }
}

[[noreturn]] void bad(const std::string &text) { throw std::invalid_argument(text); }

int elem_size(LitniceView t) { return t->dtype == LITNICE_B200_VIEW_BF16 ? 2 : 4; }

void check_tensor(LitniceView t, const char *name, uint32_t rank, bool bf16_too) {
  const std::string n(name);
  if (t == nullptr) bad(n + " is a null view");
  if (t->data == nullptr) bad(n + " has a null data pointer");
  if (t->device != 1u) bad(n + " is not on the GPU");
  if (t->dtype != LITNICE_B200_VIEW_F32 && !(bf16_too && t->dtype == LITNICE_B200_VIEW_BF16))
    bad(n + (bf16_too ? " is neither f32 nor bfloat16" : " is not f32"));
  if (rank != 0 ? t->rank != rank : t->rank < 2 || t->rank > LITNICE_TENSOR_MAX_RANK)
    bad(n + " has rank " + std::to_string(t->rank));
  const int size = elem_size(t);
  if (reinterpret_cast<uintptr_t>(t->data) % size) bad(n + " does not lie on an element boundary");
  for (uint32_t i = 0; i < t->rank; ++i) {
    if (t->dims[i] <= 0 || t->dims[i] > MAX_EXTENT) bad(n + " has an extent of " + std::to_string(t->dims[i]));
    if (t->strides_bytes[i] % size) bad(n + " has a stride that is no multiple of its element");
    if (t->dims[i] > 1 && (t->strides_bytes[i] > (1ll << 50) || t->strides_bytes[i] < -(1ll << 50))) bad(n + " has an impossible stride");
  }
}

// Elements of a result do not lie on one another: its axes, by stride, each step over all of the one below.
void check_result(LitniceView t, const char *name) {
  int order[LITNICE_TENSOR_MAX_RANK], k = 0;
  for (uint32_t i = 0; i < t->rank; ++i)
    if (t->dims[i] > 1) order[k++] = (int)i;
  for (int i = 1; i < k; ++i)
    for (int j = i; j > 0 && std::llabs(t->strides_bytes[order[j]]) < std::llabs(t->strides_bytes[order[j - 1]]); --j)
      std::swap(order[j], order[j - 1]);
  __int128 reach = elem_size(t);
  for (int i = 0; i < k; ++i) {
    const long long s = std::llabs(t->strides_bytes[order[i]]);
    if ((__int128)s < reach) bad(std::string(name) + " is a result whose elements overlap");
    reach = (__int128)s * (t->dims[order[i]] - 1) + reach;
  }
}

void check_like(LitniceView t, LitniceView u, const char *name, const char *other) {
  bool same = t->dtype == u->dtype && t->rank == u->rank;
  for (uint32_t i = 0; same && i < t->rank; ++i) same = t->dims[i] == u->dims[i];
  if (!same) bad(std::string(name) + " differs from " + other + " in shape or type");
}

// A result (or the workspace) that begins where another argument does would change it under the kernels. (Slices of one buffer may
// interleave: what begins elsewhere is the caller's care.)
struct Named {
  const void *p;
  const char *name;
  Named(const void *at, const char *n) : p(at), name(n) {}
  Named(LitniceView t, const char *n) : p(t ? t->data : nullptr), name(n) {}
};
void check_apart(Named result, std::initializer_list<Named> others) {
  for (const Named &o : others)
    if (o.p != nullptr && result.p == o.p) bad(std::string(result.name) + " lies on " + o.name);
}

void check_workspace(const void *workspace, uint64_t have, uint64_t need) {
  if (workspace == nullptr) bad("null workspace");
  if (reinterpret_cast<uintptr_t>(workspace) % 256) bad("the workspace is not on a 256-byte boundary");
  if (have < need) bad("the workspace has " + std::to_string(have) + " bytes, " + std::to_string(need) + " are needed");
}

void check_floats(const void *p, const char *name) {
  if (p == nullptr) bad(std::string(name) + " is null");
  if (reinterpret_cast<uintptr_t>(p) % 4) bad(std::string(name) + " does not lie on an element boundary");
}

HeadView head_view(LitniceView t) {
  const int size = elem_size(t);
  HeadView v;
  v.p = static_cast<char *>(t->data);
  long long s[4];
  for (int i = 0; i < 4; ++i) s[i] = t->dims[i] > 1 ? t->strides_bytes[i] / size : 0;
  v.s = s[0];
  v.r = s[1];
  v.h = s[2];
  v.c = t->dims[3] > 1 ? s[3] : 1;
  return v;
}

TrainAttention attention_args(LitniceView q, LitniceView k, LitniceView v, const litnice_b200_attention_options *o) {
  check_tensor(q, "q", 4, true);
  check_tensor(k, "k", 4, true);
  check_tensor(v, "v", 4, true);
  check_like(v, k, "v", "k");
  if (k->dtype != q->dtype) bad("k differs from q in type");
  if (k->dims[0] != q->dims[0]) bad("k has another number of streams than q");
  if (k->dims[3] != q->dims[3]) bad("k has another head dimension than q");
  if (q->dims[3] > TRAIN_MAX_DIM) bad("heads of more than " + std::to_string(TRAIN_MAX_DIM) + " dimensions");
  if (q->dims[2] % k->dims[2]) bad("the query heads are no multiple of the key heads");
  if (o == nullptr) bad("null options");
  if (!std::isfinite(o->scale)) bad("the scale is not finite");
  if (o->first < 0 || o->first + q->dims[1] > MAX_EXTENT) bad("first is out of range");
  if (o->window < 0 || o->window > MAX_EXTENT) bad("the window is out of range");
  if (o->lengths != nullptr && reinterpret_cast<uintptr_t>(o->lengths) % 4) bad("lengths do not lie on an element boundary");
  TrainAttention a;
  a.q = head_view(q);
  a.k = head_view(k);
  a.v = head_view(v);
  a.lengths = o->lengths;
  a.streams = (int)q->dims[0];
  a.n = (int)q->dims[1];
  a.heads = (int)q->dims[2];
  a.dim = (int)q->dims[3];
  a.m = (int)k->dims[1];
  a.groups = (int)k->dims[2];
  a.scale = o->scale;
  a.causal = o->causal != 0;
  a.first = o->first;
  a.window = o->window;
  a.seen = a.causal && a.first + a.n < a.m ? a.first + a.n : a.m;
  a.bf16 = q->dtype == LITNICE_B200_VIEW_BF16;
  if ((__int128)a.streams * a.heads * a.n > (__int128)1 << 40 || (__int128)a.streams * a.groups * a.m > (__int128)1 << 40)
    bad("too many rows, heads and streams for one call");
  return a;
}

// Bytes in front of the operands' parts: delta of a backward pass.
uint64_t delta_bytes(LitniceView q) { return ((uint64_t)q->dims[0] * (uint64_t)q->dims[1] * (uint64_t)q->dims[2] * 4 + 255) / 256 * 256; }

uint64_t attention_workspace(LitniceView q, LitniceView k, bool backward) {
  if (k->dims[0] != q->dims[0]) bad("k has another number of streams than q");
  uint64_t need = 256 + (backward ? delta_bytes(q) : 0);
  if (q->dtype != LITNICE_B200_VIEW_BF16)
    need += train_attention_f32_workspace(q->dims[0], q->dims[1], k->dims[1], q->dims[2], k->dims[2], q->dims[3], backward);
  return need;
}

void muon_sizes(LitniceView t) {
  const long long m = t->dims[t->rank - 2], n = t->dims[t->rank - 1];
  __int128 count = 1;
  for (uint32_t i = 0; i + 2 < t->rank; ++i) count *= t->dims[i];
  if (count > 65535) bad("more than 65535 matrices in one call");
  if ((m < n ? m : n) > 32768 || (m < n ? n : m) > (1 << 22)) bad("a matrix of " + std::to_string(m) + " x " + std::to_string(n));
  if (count * ((m + 127) / 128) * ((n + 127) / 128) > 0x3fffffff) bad("too many matrices of this size for one call");
}

uint64_t muon_workspace(LitniceView t) {
  long long count = 1;
  for (uint32_t i = 0; i + 2 < t->rank; ++i) count *= t->dims[i];
  return muon_workspace_bytes(count, t->dims[t->rank - 2], t->dims[t->rank - 1]);
}

}  // namespace

extern "C" {

int litnice_b200_attention_forward(LitniceView q, LitniceView k, LitniceView v, const litnice_b200_attention_options *options,
                                   LitniceView out, float *lse, void *workspace, uint64_t workspace_bytes, void *stream) {
  return guarded("attention_forward", [&] {
    TrainAttention a = attention_args(q, k, v, options);
    check_tensor(out, "out", 4, true);
    check_like(out, q, "out", "q");
    check_result(out, "out");
    check_floats(lse, "lse");
    check_workspace(workspace, workspace_bytes, attention_workspace(q, k, false));
    const Named lengths{options->lengths, "lengths"};
    check_apart({out, "out"}, {{q, "q"}, {k, "k"}, {v, "v"}, lengths});
    check_apart({lse, "lse"}, {{q, "q"}, {k, "k"}, {v, "v"}, {out, "out"}, lengths});
    check_apart({workspace, "the workspace"}, {{q, "q"}, {k, "k"}, {v, "v"}, {out, "out"}, {lse, "lse"}, lengths});
    a.out = head_view(out);
    a.lse = lse;
    launch_train_attention_forward(a, workspace, static_cast<cudaStream_t>(stream));
  });
}

uint64_t litnice_b200_attention_forward_workspace(LitniceView q, LitniceView k) {
  uint64_t need = 0;
  guarded("attention_forward_workspace", [&] {
    check_tensor(q, "q", 4, true);
    check_tensor(k, "k", 4, true);
    need = attention_workspace(q, k, false);
  });
  return need;
}

uint64_t litnice_b200_attention_backward_workspace(LitniceView q, LitniceView k) {
  uint64_t need = 0;
  guarded("attention_backward_workspace", [&] {
    check_tensor(q, "q", 4, true);
    check_tensor(k, "k", 4, true);
    need = attention_workspace(q, k, true);
  });
  return need;
}

int litnice_b200_attention_backward(LitniceView dout, LitniceView q, LitniceView k, LitniceView v, LitniceView out,
                                    const float *lse, const litnice_b200_attention_options *options, LitniceView dq,
                                    LitniceView dk, LitniceView dv, void *workspace, uint64_t workspace_bytes, void *stream) {
  return guarded("attention_backward", [&] {
    TrainAttention a = attention_args(q, k, v, options);
    check_tensor(dout, "dout", 4, true);
    check_tensor(out, "out", 4, true);
    check_tensor(dq, "dq", 4, true);
    check_tensor(dk, "dk", 4, true);
    check_tensor(dv, "dv", 4, true);
    check_like(dout, q, "dout", "q");
    check_like(out, q, "out", "q");
    check_like(dq, q, "dq", "q");
    check_like(dk, k, "dk", "k");
    check_like(dv, k, "dv", "k");
    check_result(dq, "dq");
    check_result(dk, "dk");
    check_result(dv, "dv");
    check_floats(lse, "lse");
    check_workspace(workspace, workspace_bytes, attention_workspace(q, k, true));
    const Named lengths{options->lengths, "lengths"}, sums{lse, "lse"};
    check_apart({dq, "dq"}, {{dout, "dout"}, {q, "q"}, {k, "k"}, {v, "v"}, {out, "out"}, {dk, "dk"}, {dv, "dv"}, sums, lengths});
    check_apart({dk, "dk"}, {{dout, "dout"}, {q, "q"}, {k, "k"}, {v, "v"}, {out, "out"}, {dv, "dv"}, sums, lengths});
    check_apart({dv, "dv"}, {{dout, "dout"}, {q, "q"}, {k, "k"}, {v, "v"}, {out, "out"}, sums, lengths});
    check_apart({workspace, "the workspace"}, {{dout, "dout"}, {q, "q"}, {k, "k"}, {v, "v"}, {out, "out"}, {dq, "dq"}, {dk, "dk"},
                                               {dv, "dv"}, sums, lengths});
    a.dout = head_view(dout);
    a.out = head_view(out);
    a.dq = head_view(dq);
    a.dk = head_view(dk);
    a.dv = head_view(dv);
    a.lse = const_cast<float *>(lse);
    launch_train_attention_backward(a, static_cast<float *>(workspace), static_cast<char *>(workspace) + delta_bytes(q),
                                    static_cast<cudaStream_t>(stream));
  });
}

uint64_t litnice_b200_policy_loss_workspace(LitniceView logits) {
  uint64_t need = 0;
  guarded("policy_loss_workspace", [&] {
    check_tensor(logits, "logits", 2, true);
    need = policy_loss_workspace_bytes(logits->dims[0]);
  });
  return need;
}

int litnice_b200_policy_loss(LitniceView logits, const int32_t *targets, const float *old_logp, const float *advantage,
                             const float *ref_logp, const float *weight, const litnice_b200_policy_options *options,
                             float *loss, float *logp, LitniceView dlogits, void *workspace, uint64_t workspace_bytes,
                             void *stream) {
  return guarded("policy_loss", [&] {
    check_tensor(logits, "logits", 2, true);
    if (logits->dims[1] > 1 && logits->strides_bytes[1] != elem_size(logits)) bad("the columns of logits are not contiguous");
    check_floats(targets, "targets");
    check_floats(old_logp, "old_logp");
    check_floats(advantage, "advantage");
    if (options == nullptr) bad("null options");
    if (!(options->temp > 0.f) || !std::isfinite(options->temp) || !std::isfinite(1.f / options->temp)) bad("temp is not above 0");
    if (!(options->clip_low >= 0.f && options->clip_low <= 1.f) || !(options->clip_high >= 0.f)) bad("a clip is out of range");
    if (!std::isfinite(options->kl_weight)) bad("kl_weight is not finite");
    if (options->kl_weight != 0.f) check_floats(ref_logp, "ref_logp");
    if (weight != nullptr) check_floats(weight, "weight");
    check_floats(loss, "loss");
    check_floats(logp, "logp");
    PolicyLoss a;
    a.rows = (int)logits->dims[0];
    a.vocab = (int)logits->dims[1];
    a.bf16 = logits->dtype == LITNICE_B200_VIEW_BF16;
    a.logits = static_cast<const char *>(logits->data);
    a.ld = a.rows > 1 ? logits->strides_bytes[0] / elem_size(logits) : 0;
    if (dlogits != nullptr) {
      check_tensor(dlogits, "dlogits", 2, true);
      check_like(dlogits, logits, "dlogits", "logits");
      check_result(dlogits, "dlogits");
      if (dlogits->dims[1] > 1 && dlogits->strides_bytes[1] != elem_size(dlogits)) bad("the columns of dlogits are not contiguous");
      a.dlogits = static_cast<char *>(dlogits->data);
      a.dld = a.rows > 1 ? dlogits->strides_bytes[0] / elem_size(dlogits) : 0;
      if (a.dlogits == a.logits && a.dld != a.ld) bad("dlogits lies on logits with another stride");
    }
    check_workspace(workspace, workspace_bytes, policy_loss_workspace_bytes(a.rows));
    const Named inputs[] = {{targets, "targets"}, {old_logp, "old_logp"}, {advantage, "advantage"}, {ref_logp, "ref_logp"}, {weight, "weight"}};
    const Named results[] = {{loss, "loss"}, {logp, "logp"}, {dlogits, "dlogits"}, {workspace, "the workspace"}};
    for (int i = 0; i < 4; ++i) {
      if (results[i].p == nullptr) continue;
      for (const Named &input : inputs) check_apart(results[i], {input});
      if (i != 2) check_apart(results[i], {{logits, "logits"}});  // (the gradient may take its place)
      for (int j = 0; j < i; ++j) check_apart(results[i], {results[j]});
    }
    a.targets = targets;
    a.old_logp = old_logp;
    a.advantage = advantage;
    a.ref_logp = ref_logp;
    a.weight = weight;
    a.loss = loss;
    a.logp = logp;
    a.inv_temp = 1.f / options->temp;
    a.clip_low = options->clip_low;
    a.clip_high = options->clip_high;
    a.kl_weight = options->kl_weight;
    launch_policy_loss(a, workspace, static_cast<cudaStream_t>(stream));
  });
}

uint64_t litnice_b200_orthogonalise_workspace(LitniceView x) {
  uint64_t need = 0;
  guarded("orthogonalise_workspace", [&] {
    check_tensor(x, "x", 0, false);
    muon_sizes(x);
    need = muon_workspace(x);
  });
  return need;
}

int litnice_b200_orthogonalise(LitniceView x, LitniceView out, int32_t steps, void *workspace, uint64_t workspace_bytes,
                               void *stream) {
  return guarded("orthogonalise", [&] {
    check_tensor(x, "x", 0, false);
    check_tensor(out, "out", 0, false);
    check_like(out, x, "out", "x");
    check_result(out, "out");
    muon_sizes(x);
    if (steps < 0 || steps > 100) bad("steps is out of range");
    check_workspace(workspace, workspace_bytes, muon_workspace(x));
    check_apart({workspace, "the workspace"}, {{x, "x"}, {out, "out"}});
    // (in place, a matrix is read whole before it is written; another matrix of the call may not have been)
    for (uint32_t i = 0; out->data == x->data && i < x->rank; ++i)
      if (x->dims[i] > 1 && out->strides_bytes[i] != x->strides_bytes[i]) bad("out lies on x with another stride");
    MuonStep g;
    g.grads = make_mat_view(x, "x");
    g.params = make_mat_view(out, "out");
    g.steps = steps;
    launch_muon(g, workspace, static_cast<cudaStream_t>(stream));
  });
}

int litnice_b200_muon_step(LitniceView params, LitniceView grads, LitniceView momentum, const litnice_b200_muon_options *options,
                           void *workspace, uint64_t workspace_bytes, void *stream) {
  return guarded("muon_step", [&] {
    check_tensor(params, "params", 0, false);
    check_tensor(grads, "grads", 0, false);
    check_tensor(momentum, "momentum", 0, false);
    check_like(params, grads, "params", "grads");
    check_like(momentum, grads, "momentum", "grads");
    check_result(params, "params");
    check_result(momentum, "momentum");
    muon_sizes(grads);
    if (options == nullptr) bad("null options");
    if (options->steps < 0 || options->steps > 100) bad("steps is out of range");
    if (!std::isfinite(options->lr) || !std::isfinite(options->mu) || !std::isfinite(options->weight_decay))
      bad("an option is not finite");
    check_workspace(workspace, workspace_bytes, muon_workspace(grads));
    check_apart({params, "params"}, {{grads, "grads"}, {momentum, "momentum"}});
    check_apart({momentum, "momentum"}, {{grads, "grads"}});
    check_apart({workspace, "the workspace"}, {{params, "params"}, {grads, "grads"}, {momentum, "momentum"}});
    MuonStep g;
    g.step = 1;
    g.grads = make_mat_view(grads, "grads");
    g.momentum = make_mat_view(momentum, "momentum");
    g.params = make_mat_view(params, "params");
    g.lr = options->lr;
    g.mu = options->mu;
    g.weight_decay = options->weight_decay;
    g.nesterov = options->nesterov != 0;
    g.steps = options->steps;
    launch_muon(g, workspace, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"

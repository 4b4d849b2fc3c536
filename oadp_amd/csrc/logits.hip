// logits.hip — operators on rows of logits: log probabilities of given tokens with the entropy, the log of the
// partition sum and the top alternatives; a student's distillation loss against a teacher's top logits; the gradients
// of both.  The C entry points are at the end of the file (include/oake_hip.h states what they compute).
//
// A row of `vocab` logits x (fp32, fp16 or bf16) and a positive scale give z = scale * x and p = softmax(z).  Everything
// is kept relative to the row's largest logit m: d = scale * (x - m) <= 0, S = sum e^d, so that log p = d - log S keeps
// its digits where it is small, whatever the size of m (lse = scale * m + log S is rounded once, at the end).  All of it
// is fp32; 16 bits appear only in the logits and, rounded once, in their gradient.
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/oake_hip.h"
#include "common.h"
#include "kernels.h"

namespace oake {
namespace {

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kThreads = 256;
constexpr int kMaxTop = 128;     // entries of a list of alternatives
constexpr int kMaxList = 1024;   // given tokens of a row / entries of a teacher's list

// Sort key of a logit: unsigned order = value order, -0 and +0 equal, every NaN above every number (torch.sort's
// order).  kKeyNegInf and below: no alternative (masked, or probability zero).
constexpr uint32_t kKeyNegInf = 0x007FFFFFu, kKeyNan = 0xFFFFFFFEu;  // (no key is ~0: "above all")
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return kKeyNan;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// ... with the place: the larger key is the better alternative, of equal logits the lowest index
__device__ __forceinline__ uint64_t place_key(float x, uint32_t j) {
  return (uint64_t)order_key(x) << 32 | (0xFFFFFFFFu - j);
}

struct Rows {  // rows of logits and what of them is allowed
  const void* x;
  int64_t rows, vocab, stride;
  const uint8_t* mask;   // nullptr: everything; else 1 byte a logit, 0 = not allowed
  int64_t mask_stride;   // 0: one mask for all rows
  float scale;
};
template <typename T>
__device__ __forceinline__ float logit(const T* x, const uint8_t* mask, int64_t j) {
  return mask && !mask[j] ? -kInf : (float)x[j];
}

__device__ __forceinline__ int64_t load_id(const void* ids, int wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(ids)[i] : (int64_t)static_cast<const int32_t*>(ids)[i];
}

// ---- reductions over the block ------------------------------------------------------------------------------
template <typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, Op op, V* tmp) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o, 64));
  __syncthreads();  // (tmp may still be read from the reduction before)
  if (threadIdx.x % 64 == 0) tmp[threadIdx.x / 64] = v;
  __syncthreads();
  v = tmp[0];
  for (int w = 1; w < kThreads / 64; ++w) v = op(v, tmp[w]);
  return v;
}
struct Add {
  template <typename V>
  __device__ V operator()(V a, V b) const { return a + b; }
};
struct Max {
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
  __device__ uint64_t operator()(uint64_t a, uint64_t b) const { return a > b ? a : b; }
};
union Tmp {
  float f[kThreads / 64];
  double d[kThreads / 64];
  uint64_t u[kThreads / 64];
};

// log p of one place, given its logit: -inf where the row holds nothing there
__device__ __forceinline__ float logp_at(float x, float m, float log_s, float scale) {
  return x == -kInf && log_s == log_s ? -kInf : (x - m) * scale - log_s;
}

// ---- token_logprobs -----------------------------------------------------------------------------------------
struct ScoreArgs {
  Rows r;
  const void* targets;
  int wide_ids, n_targets, top;
  float *logprobs, *lse, *entropy, *top_logprobs, *stats;
  int64_t* top_indices;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void score_kernel(ScoreArgs a) {
  __shared__ Tmp tmp;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.r.x) + row * a.r.stride;
  const uint8_t* mask = a.r.mask ? a.r.mask + row * a.r.mask_stride : nullptr;
  const float c = a.r.scale * kLog2e;
  float m = -kInf;
  for (int64_t j = threadIdx.x; j < a.r.vocab; j += kThreads) m = fmaxf(m, logit(x, mask, j));
  m = block_reduce(m, Max{}, tmp.f);
  if (m == -kInf) m = 0.f;  // nothing allowed (the sum is 0), or nothing but NaN (the sum is NaN)
  float s = 0.f, t = 0.f;
  for (int64_t j = threadIdx.x; j < a.r.vocab; j += kThreads) {
    const float d = (logit(x, mask, j) - m) * c, e = __builtin_amdgcn_exp2f(d);
    s += e;
    t += e * fmaxf(d, -200.f);  // 2^-200 is 0 in fp32: a place of probability zero adds 0, not 0 * inf
  }
  s = block_reduce(s, Add{}, tmp.f);
  t = block_reduce(t, Add{}, tmp.f);
  const bool empty = s == 0.f;
  const float log_s = empty ? -kInf : logf(s);
  const float h = empty ? 0.f : log_s - t * kLn2 / s;
  if (threadIdx.x == 0) {
    if (a.lse) a.lse[row] = empty ? -kInf : m * a.r.scale + log_s;
    if (a.entropy) a.entropy[row] = h;
    if (a.stats) {
      a.stats[row * 4 + 0] = m;
      a.stats[row * 4 + 1] = log_s;
      a.stats[row * 4 + 2] = h;
      a.stats[row * 4 + 3] = 0.f;
    }
  }
  for (int i = threadIdx.x; i < a.n_targets; i += kThreads) {
    const int64_t j = load_id(a.targets, a.wide_ids, row * a.n_targets + i);
    a.logprobs[row * a.n_targets + i] = j < 0               ? 0.f
                                        : j >= a.r.vocab ? __builtin_nanf("")
                                                            : logp_at(logit(x, mask, j), m, log_s, a.r.scale);
  }
  uint64_t last = ~0ull;
  for (int i = 0; i < a.top; ++i) {
    uint64_t best = 0;
    for (int64_t j = threadIdx.x; j < a.r.vocab; j += kThreads) {
      const uint64_t k = place_key(logit(x, mask, j), (uint32_t)j);
      if (k < last && k > best) best = k;
    }
    last = block_reduce(best, Max{}, tmp.u);
    if (threadIdx.x == 0) {
      const bool some = (uint32_t)(last >> 32) > kKeyNegInf;
      const int64_t j = some ? 0xFFFFFFFFu - (uint32_t)last : 0;
      a.top_indices[row * a.top + i] = some ? j : -1;
      a.top_logprobs[row * a.top + i] = some ? logp_at((float)x[j], m, log_s, a.r.scale) : -kInf;
    }
  }
}

// ---- the teacher's list of one row ----------------------------------------------------------------------------
struct TeacherArgs {
  const void* ids;
  const float* v;
  int wide_ids, n, tail;
};
struct Teacher {       // (in LDS)
  int id[kMaxList];    // -1: absent
  float v[kMaxList], q[kMaxList];
  float q_sum, q_rest, log_norm;  // sum of q; the bucket's probability; log q = v - log_norm
  bool some;                      // there is an entry at all
};

// q of a row: the softmax of its entries, or (tail) e^v as they are and a bucket for what is left of 1.  The bucket is a
// difference from 1, taken in 64 bits.  An id that the vocabulary does not have makes the row NaN.
__device__ __forceinline__ void teacher_row(const TeacherArgs& a, int64_t row, int64_t vocab, Teacher& s, Tmp& tmp) {
  float best = -kInf, some = 0.f;
  for (int i = threadIdx.x; i < a.n; i += kThreads) {
    const int64_t j = load_id(a.ids, a.wide_ids, row * a.n + i);
    float v = a.v[row * a.n + i];
    if (j < 0) v = -kInf;
    if (j >= vocab && v != -kInf) v = __builtin_nanf("");
    s.id[i] = v == -kInf || j >= vocab ? -1 : (int)j;
    s.v[i] = v;
    best = fmaxf(best, v);
    if (v != -kInf) some = 1.f;
  }
  best = block_reduce(best, Max{}, tmp.f);
  some = block_reduce(some, Max{}, tmp.f);
  if (a.tail || best == -kInf) best = 0.f;  // (no entry: every q is 0)
  double sum = 0;
  for (int i = threadIdx.x; i < a.n; i += kThreads) sum += exp((double)(s.v[i] - best));
  sum = block_reduce(sum, Add{}, tmp.d);
  const float log_norm = a.tail || sum == 0 ? best : best + (float)log(sum);
  float q_sum = 0.f;
  for (int i = threadIdx.x; i < a.n; i += kThreads) {
    const float q = a.tail || sum == 0 ? expf(s.v[i]) : expf(s.v[i] - best) / (float)sum;
    s.q[i] = q;
    q_sum += q;
  }
  q_sum = block_reduce(q_sum, Add{}, tmp.f);
  if (threadIdx.x == 0) {
    s.q_sum = q_sum;
    s.q_rest = a.tail ? (float)(sum > 1 ? 0 : 1 - sum) : 0.f;
    s.log_norm = log_norm;
    s.some = some != 0.f;
  }
  __syncthreads();
}
__device__ __forceinline__ bool listed(const Teacher& s, int n, int64_t j) {
  for (int i = 0; i < n; ++i)
    if (s.id[i] == j) return true;
  return false;
}

struct DistillArgs {
  Rows r;
  TeacherArgs t;
  float *loss, *stats;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_kernel(DistillArgs a) {
  __shared__ Tmp tmp;
  __shared__ Teacher te;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.r.x) + row * a.r.stride;
  const float c = a.r.scale * kLog2e;
  teacher_row(a.t, row, a.r.vocab, te, tmp);
  if (!te.some) {  // no teacher: no loss (the backward pass reads the list again, and no statistics)
    if (threadIdx.x == 0) a.loss[row] = 0.f;
    return;
  }
  float m = -kInf, mo = -kInf;  // all places; the places outside the list
  for (int64_t j = threadIdx.x; j < a.r.vocab; j += kThreads) {
    const float v = (float)x[j];
    m = fmaxf(m, v);
    if (a.t.tail && !listed(te, a.t.n, j)) mo = fmaxf(mo, v);
  }
  m = block_reduce(m, Max{}, tmp.f);
  mo = block_reduce(mo, Max{}, tmp.f);
  if (m == -kInf) m = 0.f;
  if (mo == -kInf) mo = 0.f;
  float s = 0.f, so = 0.f;
  for (int64_t j = threadIdx.x; j < a.r.vocab; j += kThreads) {
    const float v = (float)x[j];
    s += __builtin_amdgcn_exp2f((v - m) * c);
    if (a.t.tail && !listed(te, a.t.n, j)) so += __builtin_amdgcn_exp2f((v - mo) * c);
  }
  s = block_reduce(s, Add{}, tmp.f);
  so = block_reduce(so, Add{}, tmp.f);
  const float log_s = s == 0.f ? -kInf : logf(s), log_so = so == 0.f ? -kInf : logf(so);
  float loss = 0.f;
  for (int i = threadIdx.x; i < a.t.n; i += kThreads)
    if (te.q[i] != 0.f) {
      const float lp = te.id[i] < 0 ? 0.f : logp_at((float)x[te.id[i]], m, log_s, a.r.scale);
      loss += te.q[i] * (te.v[i] - te.log_norm - lp);
    }
  loss = block_reduce(loss, Add{}, tmp.f);
  if (threadIdx.x == 0) {
    const float rest = log_so == -kInf ? 0.f : te.q_rest;
    if (rest != 0.f) loss += rest * (logf(rest) - ((mo - m) * a.r.scale + log_so - log_s));
    a.loss[row] = loss;
    a.stats[row * 8 + 0] = m;
    a.stats[row * 8 + 1] = log_s;
    a.stats[row * 8 + 2] = mo;
    a.stats[row * 8 + 3] = log_so;
  }
}

// ---- gradients --------------------------------------------------------------------------------------------------
// Both operators' gradients are, over the whole row, p'_j * (a0 + a1 * (log p_j + H)) with p' = e^(d' - log S'), and at
// the few listed places j (given tokens and alternatives; the teacher's list) b0 * p_j + ... plus the weights of the
// entries that name j.  The row is written first, then the listed places again, each by the first entry that names it
// with the weights of all of them, so that no sum depends on an order.
template <typename T>
__device__ __forceinline__ void fill(T* g, int64_t n, float v) {
  for (int64_t j = threadIdx.x; j < n; j += kThreads) g[j] = to16<T>(v);
}

struct ScoreGradArgs {
  Rows r;
  const void* targets;
  int wide_ids, n_targets, top;
  const int64_t* top_indices;
  const float *stats, *g_logprobs, *g_lse, *g_entropy, *g_top;
  void* grad;
  int64_t grad_stride;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void score_grad_kernel(ScoreGradArgs a) {
  __shared__ Tmp tmp;
  __shared__ int id[kMaxList + kMaxTop];
  __shared__ float w[kMaxList + kMaxTop];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.r.x) + row * a.r.stride;
  const uint8_t* mask = a.r.mask ? a.r.mask + row * a.r.mask_stride : nullptr;
  T* g = static_cast<T*>(a.grad) + row * a.grad_stride;
  const float m = a.stats[row * 4], log_s = a.stats[row * 4 + 1], h = a.stats[row * 4 + 2];
  if (log_s == -kInf) return fill(g, a.r.vocab, 0.f);
  const int nt = a.g_logprobs ? a.n_targets : 0, n = nt + (a.g_top ? a.top : 0);
  float sum = 0.f;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int64_t j = i < nt ? load_id(a.targets, a.wide_ids, row * a.n_targets + i) : a.top_indices[row * a.top + i - nt];
    float v = i < nt ? a.g_logprobs[row * a.n_targets + i] : a.g_top[row * a.top + i - nt];
    if (j < 0) v = 0.f;                                              // padding
    else if (j >= a.r.vocab) v = __builtin_nanf("");                // (its log probability is NaN)
    else if (logit(x, mask, j) == -kInf) v = 0.f;                   // -inf whatever the logits: a constant
    id[i] = j < 0 || j >= a.r.vocab || v == 0.f ? -1 : (int)j;
    w[i] = v;
    sum += v;
  }
  sum = block_reduce(sum, Add{}, tmp.f);
  const float gh = a.g_entropy ? a.g_entropy[row] : 0.f;
  const float a0 = (a.g_lse ? a.g_lse[row] : 0.f) - sum;
  const float scale = a.r.scale;
  const auto dense = [&](float v) {  // dH / dz_j = -p_j (log p_j + H)
    const float lp = fmaxf((v - m) * scale - log_s, -150.f);
    return __builtin_amdgcn_exp2f((v - m) * (scale * kLog2e) - log_s * kLog2e) * (a0 - gh * (lp + h));
  };
  for (int64_t j = threadIdx.x; j < a.r.vocab; j += kThreads)
    g[j] = to16<T>(mask && !mask[j] ? 0.f : dense((float)x[j]) * scale);
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    if (id[i] < 0) continue;
    float v = 0.f;
    bool first = true;
    for (int k = 0; k < n; ++k)
      if (id[k] == id[i]) {
        first = first && k >= i;
        v += w[k];
      }
    if (first) g[id[i]] = to16<T>((dense((float)x[id[i]]) + v) * scale);
  }
}

struct DistillGradArgs {
  Rows r;
  TeacherArgs t;
  const float *stats, *g_loss;
  void* grad;
  int64_t grad_stride;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_grad_kernel(DistillGradArgs a) {
  __shared__ Tmp tmp;
  __shared__ Teacher te;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.r.x) + row * a.r.stride;
  T* g = static_cast<T*>(a.grad) + row * a.grad_stride;
  teacher_row(a.t, row, a.r.vocab, te, tmp);
  if (!te.some) return fill(g, a.r.vocab, 0.f);
  const float m = a.stats[row * 8], log_s = a.stats[row * 8 + 1], mo = a.stats[row * 8 + 2], log_so = a.stats[row * 8 + 3];
  if (log_s == -kInf) return fill(g, a.r.vocab, 0.f);
  const float up = a.g_loss[row] * a.r.scale, c = a.r.scale * kLog2e;
  const bool tail = a.t.tail && log_so != -kInf;
  const float rest = tail ? te.q_rest : 0.f, q_all = te.q_sum + rest;
  // outside the list: p_j q_all - rest e^(z_j - lse_o) = e^(z_j - lse_o) (p_o q_all - rest), p_o the student's bucket
  const float ref = tail ? mo : m, log_ref = (tail ? log_so : log_s) * kLog2e;
  const float p_o = tail ? expf((mo - m) * a.r.scale + log_so - log_s) : 1.f;
  const float a0 = up * (p_o * q_all - rest);
  for (int64_t j = threadIdx.x; j < a.r.vocab; j += kThreads)
    g[j] = to16<T>(a0 * __builtin_amdgcn_exp2f(((float)x[j] - ref) * c - log_ref));
  __syncthreads();
  for (int i = threadIdx.x; i < a.t.n; i += kThreads) {
    if (te.id[i] < 0) continue;
    float q = 0.f;
    bool first = true;
    for (int k = 0; k < a.t.n; ++k)
      if (te.id[k] == te.id[i]) {
        first = first && k >= i;
        q += te.q[k];
      }
    const float p = __builtin_amdgcn_exp2f(((float)x[te.id[i]] - m) * c - log_s * kLog2e);
    if (first) g[te.id[i]] = to16<T>(up * (p * q_all - q));
  }
}

// ---- host side ----------------------------------------------------------------------------------------------------
__attribute__((format(printf, 2, 3))) int refuse(int code, const char* fmt, ...) {
  char text[256];
  va_list ap;
  va_start(ap, fmt);
  std::vsnprintf(text, sizeof(text), fmt, ap);
  va_end(ap);
  return fail_without_handle(code, text);
}
size_t element_size(int dtype) { return dtype == OAKE_F32 ? 4 : 2; }

int check_rows(const char* what, const void* x, int dtype, int64_t rows, int64_t vocab, int64_t stride, float scale) {
  if (dtype != OAKE_F32 && dtype != OAKE_F16 && dtype != OAKE_BF16)
    return refuse(OAKE_ERR_INVALID, "%s: the logits must be F32, F16 or BF16", what);
  if (rows < 0 || rows > INT32_MAX || vocab < 1 || vocab > INT32_MAX)
    return refuse(OAKE_ERR_INVALID, "%s: rows must be 0 .. 2^31 - 1 and vocab 1 .. 2^31 - 1", what);
  if (stride < 0) return refuse(OAKE_ERR_INVALID, "%s: a row stride is negative", what);
  if (!(scale > 0.f) || scale > 3.0e38f) return refuse(OAKE_ERR_INVALID, "%s: scale must be positive and finite", what);
  if (rows > 0 && !x) return refuse(OAKE_ERR_INVALID, "%s: null pointer", what);
  if ((uintptr_t)x % element_size(dtype)) return refuse(OAKE_ERR_INVALID, "%s: the logits are not aligned to their type", what);
  return OAKE_OK;
}
int check_list(const char* what, const char* name, const void* ids, int index_dtype, int n, int most) {
  if (n < 0 || n > most) return refuse(OAKE_ERR_INVALID, "%s: %s must be 0 .. %d", what, name, most);
  if (n && index_dtype != OAKE_I32 && index_dtype != OAKE_I64)
    return refuse(OAKE_ERR_INVALID, "%s: index_dtype must be I32 or I64", what);
  if (n && (uintptr_t)ids % (index_dtype == OAKE_I64 ? 8 : 4))
    return refuse(OAKE_ERR_INVALID, "%s: the indices are not aligned to their type", what);
  return OAKE_OK;
}
int check_grad(const char* what, void* grad, int dtype, int64_t vocab, int64_t rows, int64_t stride) {
  if (stride < vocab && rows > 1) return refuse(OAKE_ERR_INVALID, "%s: rows of the gradient overlap", what);
  if (!grad) return refuse(OAKE_ERR_INVALID, "%s: null pointer", what);
  if ((uintptr_t)grad % element_size(dtype)) return refuse(OAKE_ERR_INVALID, "%s: the gradient is not aligned to its type", what);
  return OAKE_OK;
}
int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? OAKE_OK : refuse(OAKE_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

#define OAKE_BY_TYPE(dtype, kernel, grid, s, args)                                         \
  do {                                                                                     \
    if ((dtype) == OAKE_F32) kernel<float><<<grid, kThreads, 0, s>>>(args);                \
    else if ((dtype) == OAKE_F16) kernel<f16_t><<<grid, kThreads, 0, s>>>(args);           \
    else kernel<bf16_t><<<grid, kThreads, 0, s>>>(args);                                   \
  } while (0)

}  // namespace
}  // namespace oake

using namespace oake;

extern "C" {

int oake_logits_workspace(int64_t rows, int64_t vocab, int dtype, int top, size_t* bytes) {
  const char* what = "oake_logits_workspace";
  if (!bytes) return refuse(OAKE_ERR_INVALID, "%s: null pointer", what);
  if (int rc = check_rows(what, bytes, dtype, rows, vocab, vocab, 1.f)) return rc;
  if (top < 0 || top > kMaxTop) return refuse(OAKE_ERR_INVALID, "%s: top must be 0 .. %d", what, kMaxTop);
  *bytes = 0;
  return OAKE_OK;
}

int oake_token_logprobs(const void* d_logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride, float scale,
                        const uint8_t* d_mask, int64_t mask_stride, const void* d_targets, int index_dtype, int n_targets,
                        int top, float* d_logprobs, float* d_lse, float* d_entropy, float* d_top_logprobs,
                        int64_t* d_top_indices, float* d_stats, void* d_workspace, size_t workspace_bytes, void* stream) {
  const char* what = "oake_token_logprobs";
  if (int rc = check_rows(what, d_logits, dtype, rows, vocab, row_stride, scale)) return rc;
  if (int rc = check_list(what, "n_targets", d_targets, index_dtype, n_targets, kMaxList)) return rc;
  if (top < 0 || top > kMaxTop) return refuse(OAKE_ERR_INVALID, "%s: top must be 0 .. %d", what, kMaxTop);
  if (mask_stride < 0) return refuse(OAKE_ERR_INVALID, "%s: a row stride is negative", what);
  if (rows == 0) return OAKE_OK;
  if ((n_targets && (!d_targets || !d_logprobs)) || (top && (!d_top_logprobs || !d_top_indices)))
    return refuse(OAKE_ERR_INVALID, "%s: null pointer", what);
  const ScoreArgs a{{d_logits, rows, vocab, row_stride, d_mask, mask_stride, scale},
                    d_targets, index_dtype == OAKE_I64, n_targets, top,
                    d_logprobs, d_lse, d_entropy, d_top_logprobs, d_stats, d_top_indices};
  OAKE_BY_TYPE(dtype, score_kernel, (unsigned)rows, (hipStream_t)stream, a);
  return launched(what);
}

int oake_token_logprobs_backward(const void* d_logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                                 float scale, const uint8_t* d_mask, int64_t mask_stride, const void* d_targets,
                                 int index_dtype, int n_targets, const int64_t* d_top_indices, int top,
                                 const float* d_stats, const float* d_grad_logprobs, const float* d_grad_lse,
                                 const float* d_grad_entropy, const float* d_grad_top, void* d_grad, int64_t grad_stride,
                                 void* stream) {
  const char* what = "oake_token_logprobs_backward";
  if (int rc = check_rows(what, d_logits, dtype, rows, vocab, row_stride, scale)) return rc;
  if (int rc = check_list(what, "n_targets", d_targets, index_dtype, n_targets, kMaxList)) return rc;
  if (int rc = check_list(what, "top", d_top_indices, OAKE_I64, top, kMaxTop)) return rc;
  if (mask_stride < 0) return refuse(OAKE_ERR_INVALID, "%s: a row stride is negative", what);
  if (rows == 0) return OAKE_OK;
  if (int rc = check_grad(what, d_grad, dtype, vocab, rows, grad_stride)) return rc;
  if (!d_stats || (d_grad_logprobs && n_targets && !d_targets) || (d_grad_top && top && !d_top_indices))
    return refuse(OAKE_ERR_INVALID, "%s: null pointer", what);
  const ScoreGradArgs a{{d_logits, rows, vocab, row_stride, d_mask, mask_stride, scale},
                        d_targets, index_dtype == OAKE_I64, n_targets, top, d_top_indices,
                        d_stats, d_grad_logprobs, d_grad_lse, d_grad_entropy, d_grad_top, d_grad, grad_stride};
  OAKE_BY_TYPE(dtype, score_grad_kernel, (unsigned)rows, (hipStream_t)stream, a);
  return launched(what);
}

int oake_distill_top_logits(const void* d_logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride, float scale,
                            const void* d_top_indices, int index_dtype, const float* d_top_logprobs, int top, int tail,
                            float* d_loss, float* d_stats, void* d_workspace, size_t workspace_bytes, void* stream) {
  const char* what = "oake_distill_top_logits";
  if (int rc = check_rows(what, d_logits, dtype, rows, vocab, row_stride, scale)) return rc;
  if (int rc = check_list(what, "top", d_top_indices, index_dtype, top, kMaxList)) return rc;
  if (rows == 0) return OAKE_OK;
  if (!d_loss || !d_stats || (top && (!d_top_indices || !d_top_logprobs)))
    return refuse(OAKE_ERR_INVALID, "%s: null pointer", what);
  const DistillArgs a{{d_logits, rows, vocab, row_stride, nullptr, 0, scale},
                      {d_top_indices, d_top_logprobs, index_dtype == OAKE_I64, top, tail != 0}, d_loss, d_stats};
  OAKE_BY_TYPE(dtype, distill_kernel, (unsigned)rows, (hipStream_t)stream, a);
  return launched(what);
}

int oake_distill_top_logits_backward(const void* d_logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                                     float scale, const void* d_top_indices, int index_dtype,
                                     const float* d_top_logprobs, int top, int tail, const float* d_stats,
                                     const float* d_grad_loss, void* d_grad, int64_t grad_stride, void* stream) {
  const char* what = "oake_distill_top_logits_backward";
  if (int rc = check_rows(what, d_logits, dtype, rows, vocab, row_stride, scale)) return rc;
  if (int rc = check_list(what, "top", d_top_indices, index_dtype, top, kMaxList)) return rc;
  if (rows == 0) return OAKE_OK;
  if (int rc = check_grad(what, d_grad, dtype, vocab, rows, grad_stride)) return rc;
  if (!d_stats || !d_grad_loss || (top && (!d_top_indices || !d_top_logprobs)))
    return refuse(OAKE_ERR_INVALID, "%s: null pointer", what);
  const DistillGradArgs a{{d_logits, rows, vocab, row_stride, nullptr, 0, scale},
                          {d_top_indices, d_top_logprobs, index_dtype == OAKE_I64, top, tail != 0},
                          d_stats, d_grad_loss, d_grad, grad_stride};
  OAKE_BY_TYPE(dtype, distill_grad_kernel, (unsigned)rows, (hipStream_t)stream, a);
  return launched(what);
}

}  // extern "C"

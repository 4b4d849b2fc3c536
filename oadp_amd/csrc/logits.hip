// logits.hip — operators on rows of logits: log probabilities of given tokens with the entropy, the log of the
// partition sum and the top alternatives; a student's distillation loss against a teacher's top logits; the gradients
// of both.  The C entry points are at the end of the file (include/oake_hip.h states what they compute).
//
// Each forward kernel reads the logits once and keeps them in registers for its second look (the largest first, then the
// sums relative to it), each backward kernel reads them once and writes the gradient: memory is the bound.  A copy of
// 2 x 0.54 GB reaches 5.3 TB/s on this card, 2 x 2.1 GB 4.9; a 16-bit logit at that rate leaves about 15 lane operations
// of time, so the forward kernels' instructions per logit count as well (VALU busy 0.72 in the first example below).
// Times at the kernels are of the kernel alone.
//
// A row of `vocab` logits x (fp32, fp16 or bf16) and a positive scale give z = scale * x and p = softmax(z).  Everything
// is kept relative to the row's largest logit m: d = scale * (x - m) <= 0, S = sum e^d, so that log p = d - log S keeps
// its digits where it is small, whatever the size of m (lse = scale * m + log S is rounded once, at the end).  Logits,
// exponentials, sums and gradients are fp32; the distillation loss has 64 bits where it is a difference of nearly equal
// numbers (the teacher's sum and norm, the logarithms, short rows whole); 16 bits appear only in the logits and, rounded once,
// in their gradient.
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <type_traits>

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
  bool big;              // more than the Infinity Cache holds: read past it
};
struct Split {           // a row as `parts` chunks of `chunk` places, each a workgroup's (or a wave's) own
  int64_t chunk;
  int parts;
};

__device__ __forceinline__ int64_t load_id(const void* ids, int wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(ids)[i] : (int64_t)static_cast<const int32_t*>(ids)[i];
}

// ---- 16 bytes of logits ----------------------------------------------------------------------------------------
typedef u32x4_t u32x4_any __attribute__((aligned(2)));  // at any element's address
template <typename T>
constexpr int kPer = 16 / (int)sizeof(T);
template <typename T>
constexpr int kWaveVecs = sizeof(T) == 4 ? 8 : 4;  // of a lane where a wave works on a row
constexpr int kWavePlaces = 2048;
template <typename T>
__device__ __forceinline__ float elem(u32x4_t v, int i) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(v[i]);
  else if constexpr (__is_same(T, f16_t)) return (float)__builtin_bit_cast(f16x8, v)[i];
  else return __uint_as_float(i & 1 ? v[i / 2] & 0xFFFF0000u : v[i / 2] << 16);
}
template <typename T>
__device__ __forceinline__ unsigned neg_inf_bits() {
  return sizeof(T) == 4 ? 0xFF800000u : __is_same(T, f16_t) ? 0xFC00FC00u : 0xFF80FF80u;
}
template <typename T>
__device__ __forceinline__ void drop(u32x4_t& v, int i, bool yes) {  // element i becomes -inf
  if constexpr (sizeof(T) == 4) {
    v[i] = yes ? neg_inf_bits<T>() : v[i];
  } else {
    const unsigned keep = i & 1 ? 0x0000FFFFu : 0xFFFF0000u;
    v[i / 2] = yes ? (v[i / 2] & keep) | (neg_inf_bits<T>() & ~keep) : v[i / 2];
  }
}

// x_i * c + d in one operation where the type allows (fp16: the conversion is part of v_fma_mix_f32)
template <typename T>
__device__ __forceinline__ float elem_fma(u32x4_t v, int i, float c, float d) {
  if constexpr (__is_same(T, f16_t)) {
    float r;
    if (i & 1) asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(v[i / 2]), "v"(c), "v"(d));
    else asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(v[i / 2]), "v"(c), "v"(d));
    return r;
  } else {
    return __builtin_fmaf(elem<T>(v, i), c, d);
  }
}
// The largest element.  Three at a time, or two by two in fp16, without the operations that fmaxf spends on signalling
// NaN: a vector that holds NaN may give any of its elements, or NaN.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
template <typename T>
__device__ __forceinline__ float vec_max(u32x4_t v) {
  if constexpr (sizeof(T) == 4) {
    const float a = __uint_as_float(v[0]);
    return max3(max3(a, __uint_as_float(v[1]), __uint_as_float(v[2])), __uint_as_float(v[3]), a);
  } else if constexpr (__is_same(T, f16_t)) {
    unsigned a, b;
    asm("v_pk_max_f16 %0, %1, %2" : "=v"(a) : "v"(v[0]), "v"(v[1]));
    asm("v_pk_max_f16 %0, %1, %2" : "=v"(b) : "v"(v[2]), "v"(v[3]));
    asm("v_pk_max_f16 %0, %1, %2" : "=v"(a) : "v"(a), "v"(b));
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 p = __builtin_bit_cast(f16x2, a);
    return fmaxf((float)p[0], (float)p[1]);
  } else {
    float a = max3(elem<T>(v, 0), elem<T>(v, 1), elem<T>(v, 2));
    a = max3(a, elem<T>(v, 3), elem<T>(v, 4));
    a = max3(a, elem<T>(v, 5), elem<T>(v, 6));
    return max3(a, elem<T>(v, 7), a);
  }
}

// ---- a group of NT threads: one wave of a 256-thread workgroup (NT 64), or a whole workgroup ---------------------
template <int NT>
__device__ __forceinline__ int group_tid() { return NT == 64 ? threadIdx.x % 64 : threadIdx.x; }
template <int NT>
constexpr int kBlock = NT == 64 ? 256 : NT;   // threads of a workgroup
template <int NT>
constexpr int kWaves = 4;                       // per SIMD, at least: two workgroups of 512 a CU
template <int NT>
constexpr int kGroups = NT == 64 ? 4 : 1;  // groups of a workgroup
template <int NT>
__device__ __forceinline__ int64_t group_index() {
  const int64_t b = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  return NT == 64 ? b * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : b;  // (scalar: so are the row's addresses)
}
template <int NT>
__device__ __forceinline__ void group_sync() {
  if constexpr (NT == 64) {  // LDS operations of one wave run in order: only the compiler has to keep theirs
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}

// wave reductions without LDS: rotations inside the rows of 16 lanes, then the row swaps of common.h
template <int N>
__device__ __forceinline__ float row_ror(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xF, 0xF, true));
}
__device__ __forceinline__ float wave64_sum(float v) {
  v += row_ror<8>(v);
  v += row_ror<4>(v);
  v += row_ror<2>(v);
  v += row_ror<1>(v);
  return rows16_sum(v);
}
__device__ __forceinline__ float wave64_max(float v) {
  v = fmaxf(v, row_ror<8>(v));
  v = fmaxf(v, row_ror<4>(v));
  v = fmaxf(v, row_ror<2>(v));
  v = fmaxf(v, row_ror<1>(v));
  return rows16_max(v);
}
__device__ __forceinline__ double wave64_sum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ uint64_t wave64_max(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor(v, o, 64);
    v = v > w ? v : w;
  }
  return v;
}
// over the two / eight neighbouring lanes that count for one key
__device__ __forceinline__ int sum2(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, true);  // quad_perm 1 0 3 2
}
__device__ __forceinline__ int sum8(int v) {
  v = sum2(v);
  v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, true);           // quad_perm 2 3 0 1
  return v + __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, true);  // row_half_mirror
}
template <int NT, typename V>
__device__ __forceinline__ V group_sum(V v, V* tmp) {  // tmp: NT / 64 values, free when the call begins
  v = wave64_sum(v);
  if constexpr (NT == 64) return v;
  if (threadIdx.x % 64 == 0) tmp[threadIdx.x / 64] = v;
  __syncthreads();
  v = tmp[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) v += tmp[w];
  return v;
}

// ---- a chunk of a row in the registers of a group ----------------------------------------------------------------
// The places are NV vectors of 16 bytes a thread, vector v of thread t being number v * NT + t of the chunk's, and, behind
// the last whole vector, one single value each of the first threads.  Rows of odd length put the vectors at any element's
// address: fp32 vectors lose nothing by that, 16-bit ones that begin inside a word do.  Where the loads are the bound
// (workgroups of 512) those come from the word before and move down by one element, whose place the next lane's first word
// fills - by one load for all vectors of a wave where that is another wave's, or none (shifted / as they lie, us: 2048 x 131071
// bf16, 64 alternatives 130 / 147, 4096 x 49409, 20 98 / 107; 49408 87); where instructions or stores are, they are loaded as
// they lie (65536 x 1203 fp16 69 / 67, the gradient of 65536 x 1203 69 / 64, of 2048 x 49409 70 / 67).
template <typename T, int NT, int NV>
struct Tile {
  u32x4_t v[NV];
  float single;     // -inf in the threads that have none
  int nvec, n, nv;  // whole vectors and places of the chunk; vectors that the thread's wave has any of

  // column (within the chunk) of the thread's vector v / single value
  __device__ __forceinline__ int vec_col(int vi) const { return (vi * NT + group_tid<NT>()) * kPer<T>; }
  __device__ __forceinline__ int single_col() const { return nvec * kPer<T> + group_tid<NT>(); }
  __device__ __forceinline__ bool has_single() const { return group_tid<NT>() < n - nvec * kPer<T>; }
  __device__ __forceinline__ bool has_vec(int vi) const { return vi * NT + group_tid<NT>() < nvec; }

  static constexpr bool kShift = NT == 512 && sizeof(T) == 2;

  __device__ __forceinline__ void load(const T* x, int count, bool past_cache) {
    n = count;
    nvec = n / kPer<T>;
    const int wave = NT == 64 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x) & ~63;
    nv = nvec > wave ? (nvec - wave + NT - 1) / NT : 0;
    const bool shift = kShift && (reinterpret_cast<uintptr_t>(x) & 2);
    unsigned behind = 0;  // lane vi: the last element of the wave's vectors number vi
    if (shift) {
      const int lane = threadIdx.x % 64, end = lane * NT + wave + 63;
      if (lane < nv) behind = reinterpret_cast<const unsigned short*>(x)[(end < nvec ? end : nvec - 1) * kPer<T> + kPer<T> - 1];
    }
    // (the element before an odd one is the other half of its word, and so in the same allocation)
    const u32x4_any* p = reinterpret_cast<const u32x4_any*>(x - (shift ? 1 : 0)) + group_tid<NT>();
    if (past_cache) {
#pragma unroll
      for (int vi = 0; vi < NV; ++vi)
        if (vi < nv && has_vec(vi)) {
          v[vi] = __builtin_nontemporal_load(p + vi * NT);
          asm volatile("");  // (or the compiler makes one plain access of the two)
        }
    } else {
#pragma unroll
      for (int vi = 0; vi < NV; ++vi)
        if (vi < nv && has_vec(vi)) v[vi] = p[vi * NT];
    }
    single = -kInf;
    if (has_single()) single = (float)x[single_col()];
    if (shift) {
#pragma unroll
      for (int vi = 0; vi < NV; ++vi)
        if (vi < nv) {
          const unsigned last = __builtin_amdgcn_readlane(behind, vi);
          u32x4_t q = v[vi];
          q[0] = has_vec(vi) ? q[0] : last;
          const unsigned next = __builtin_amdgcn_update_dpp((int)last, (int)q[0], 0x130, 0xF, 0xF, false);  // wave_shl:1
          q[0] = __builtin_amdgcn_alignbit(q[1], q[0], 16);
          q[1] = __builtin_amdgcn_alignbit(q[2], q[1], 16);
          q[2] = __builtin_amdgcn_alignbit(q[3], q[2], 16);
          q[3] = __builtin_amdgcn_alignbit(next, q[3], 16);
          v[vi] = q;
        }
    }
  }
  // what the mask (of the chunk's first place on) leaves out becomes -inf
  __device__ __forceinline__ void apply_mask(const uint8_t* mask) {
    typedef unsigned u32_any __attribute__((aligned(1)));
#pragma unroll
    for (int vi = 0; vi < NV; ++vi)
      if (vi < nv && has_vec(vi)) {
        const u32_any* p = reinterpret_cast<const u32_any*>(mask + vec_col(vi));
        const unsigned lo = p[0], hi = kPer<T> == 8 ? (unsigned)p[kPer<T> / 8] : 0u;
#pragma unroll
        for (int i = 0; i < kPer<T>; ++i) drop<T>(v[vi], i, ((i < 4 ? lo : hi) >> (i % 4 * 8) & 0xFF) == 0);
      }
    if (has_single() && !mask[single_col()]) single = -kInf;
  }
  // keeps the compiler from holding the unpacked values of one pass over the tile for the next
  __device__ __forceinline__ void pack() {
#pragma unroll
    for (int vi = 0; vi < NV; ++vi) asm volatile("" : "+v"(v[vi]));
  }
  // f(vector, its first column) for each of the thread's vectors
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll
    for (int vi = 0; vi < NV; ++vi)
      if (vi < nv && has_vec(vi)) f(v[vi], vi);
  }
  __device__ __forceinline__ float max() const {
    float m = single;
    each([&](u32x4_t q, int) { m = max3(m, vec_max<T>(q), m); });
    return m;
  }
};

// e_j = 2^((x_j - m) c), m the largest logit, c = scale * log2(e).  As it stands this takes two operations beside the
// exponential; x c - b with b = m c rounded takes one.  That b is off m c by r = m c - b (exact, in a fused multiply-add)
// multiplies every e_j by 2^r: p = e / S does not see it, and log S is the logarithm of S / 2^r, where 2^r is what the
// largest logit's own e came out as, so that a row of one place has log p = 0.  (Past |b| = 2^20 r would count: then the
// plain form.)
struct Ref {
  float m, c, b, r, one;
  bool fused;
  __device__ __forceinline__ Ref(float max, float c_) : m(max == -kInf ? 0.f : max), c(c_) {  // (-inf: nothing, or only NaN)
    b = m * c;
    fused = fabsf(b) < 1048576.f;
    r = fused ? __builtin_fmaf(m, c, -b) : 0.f;
    one = __builtin_amdgcn_exp2f(r);
  }
};
struct Sums {
  float s = 0.f, t = 0.f;  // sum e, sum e * log2 e
  __device__ __forceinline__ void add(float d) {
    const float e = __builtin_amdgcn_exp2f(d);
    s += e;
    t += e * fmaxf(d, -200.f);  // 2^-200 is 0 in fp32: a place of probability zero adds 0, not 0 * inf
  }
  __device__ __forceinline__ void add_finite(float d) {  // (-inf makes t NaN)
    const float e = __builtin_amdgcn_exp2f(d);
    s += e;
    t = __builtin_fmaf(e, d, t);
  }
  // From the fused form to d relative to m.  The product is rounded by itself, as that of a single place's term was (the
  // compiler would make one operation of the two): a row of one place has t = 0, entropy 0.
  __device__ __forceinline__ void relative_to_m(const Ref& ref) {
#pragma clang fp contract(off)
    const float shift = ref.r * s;
    t = (t - shift) / ref.one;
    s /= ref.one;
  }
};

// log p of one place, given its logit: -inf where the row holds nothing there
__device__ __forceinline__ float logp_at(float x, float m, float log_s, float scale) {
  return x == -kInf && log_s == log_s ? -kInf : (x - m) * scale - log_s;
}

// ---- the top alternatives -------------------------------------------------------------------------------------
// A lower bound of the row's top-th largest logit: of the maxima of (at least top) disjoint parts of the row, about the
// top-th largest - that many places reach it.  It is looked for by counting over the wave's lanes.  In the pass of the sums
// the vectors that hold a place at or above it go to LDS as they are, their places there become keys, and each key's rank is
// the number of larger ones.  49408 normal logits, top 20, of 64 parts' maxima: about 24 keys, 36 at most of 300 rows.  Where
// a list overflows (crowded equal values) or the row has NaN (which the maxima pass over), the top-th key itself is looked for
// by counting over the row.
constexpr float kLowest = -3.402823466e38f;
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ float bound_of(uint32_t prefix) {
  return prefix < 0x00800000u ? kLowest : key_value(prefix);  // (-inf is no alternative)
}
// (least, largest: of the parts; count(v): how many reach v.)  Eight halvings of the interval of values, then, where that has
// left too many parts - values of very different sizes, parts that are empty - halvings by key and by value in turn.
template <typename Count>
__device__ __forceinline__ float bound_by_count(float least, float largest, int top, Count count) {
  float lo = least, hi = largest;
  int reached = 1 << 20;
  if (least > -kInf) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float mid = 0.5f * lo + 0.5f * hi;
      const int n = count(mid);
      const bool up = n >= top;
      reached = up ? n : reached;
      lo = up ? mid : lo;
      hi = up ? hi : mid;
    }
  }
  if (reached > 2 * top + 16) {
    uint32_t a = __builtin_amdgcn_readfirstlane(order_key(lo)), b = __builtin_amdgcn_readfirstlane(order_key(hi)) + 1;
    for (int i = 0; i < 32 && b - a > 1; ++i) {
      uint32_t mid = a + (b - a) / 2;
      if (i % 2 && a > kKeyNegInf) {
        const uint32_t k = __builtin_amdgcn_readfirstlane(order_key(0.5f * key_value(a) + 0.5f * key_value(b)));
        mid = k > a && k < b ? k : mid;
      }
      const int n = count(key_value(mid));
      if (n >= top) a = mid;
      else b = mid;
      if (n >= top && n <= top + top / 8 + 2) break;
    }
    lo = a <= kKeyNegInf ? kLowest : key_value(a);
  }
  return lo;
}
template <typename Count>
__device__ __forceinline__ float bound_by_bits(int top, Count count) {
  uint32_t prefix = 0;
  for (int bit = 31; bit >= 16; --bit)
    if (count(key_value(prefix | 1u << bit)) >= top) prefix |= 1u << bit;
  return bound_of(prefix);
}
constexpr int kParts = 256;  // maxima of a workgroup's parts
template <int NT>
constexpr int kListCap = NT == 64 ? 256 : 1024;  // keys
template <int NT>
constexpr int kVecCap = NT == 64 ? 144 : 512;    // vectors that hold some

// ---- token_logprobs -----------------------------------------------------------------------------------------
struct ScoreArgs {
  Rows r;
  Split sp;
  const void* targets;
  int wide_ids, n_targets, top;
  float *logprobs, *lse, *entropy, *top_logprobs, *stats;
  int64_t* top_indices;
  float* part_sums;      // [rows, parts, 4]: m, S, sum e * log2 e of a chunk, relative to its own m
  uint64_t* part_keys;   // [rows, parts, top]: its alternatives, best first, 0 = none
};

struct RowStats {
  float m, log_s, h, inv_s;
};
// from the sums S, sum e * d (log2) relative to m
__device__ __forceinline__ RowStats row_stats(float m, float s, float t) {
  if (s == 0.f) return {m, -kInf, 0.f, 0.f};
  const float log_s = logf(s);
  return {m, log_s, log_s - fminf(t / s, 0.f) * kLn2, 1.f / s};
}
__device__ __forceinline__ void write_row(const ScoreArgs& a, int64_t row, const RowStats& st) {
  if (a.lse) a.lse[row] = st.log_s == -kInf ? -kInf : st.m * a.r.scale + st.log_s;
  if (a.entropy) a.entropy[row] = st.h;
  if (a.stats) {
    a.stats[row * 4 + 0] = st.m;
    a.stats[row * 4 + 1] = st.log_s;
    a.stats[row * 4 + 2] = st.h;
    a.stats[row * 4 + 3] = st.inv_s;
  }
}
// Given tokens: the first of each thread is fetched while the row is (its logit is two loads away), the others at the end.
template <typename T>
__device__ __forceinline__ float given_logit(const ScoreArgs& a, int64_t row, int64_t j) {  // NaN: no such token
  if (j < 0 || j >= a.r.vocab) return __builtin_nanf("");
  if (a.r.mask && !a.r.mask[row * a.r.mask_stride + j]) return -kInf;
  return (float)static_cast<const T*>(a.r.x)[row * a.r.stride + j];
}
struct Given {
  int64_t id;
  float x;
};
__device__ __forceinline__ int64_t given_id(const ScoreArgs& a, int64_t row, int i) {
  return i < a.n_targets ? load_id(a.targets, a.wide_ids, row * a.n_targets + i) : -1;
}
template <typename T>
__device__ __forceinline__ void write_given(const ScoreArgs& a, int64_t row, const RowStats& st, int t, int threads, Given g) {
  for (int i = t; i < a.n_targets; i += threads) {
    if (i != t) {
      g.id = given_id(a, row, i);
      g.x = given_logit<T>(a, row, g.id);
    }
    a.logprobs[row * a.n_targets + i] = g.id < 0 ? 0.f : logp_at(g.x, st.m, st.log_s, a.r.scale);
  }
}
__device__ __forceinline__ void write_top(const ScoreArgs& a, int64_t row, const RowStats& st, int rank, uint64_t key) {
  const bool some = (uint32_t)(key >> 32) > kKeyNegInf;
  const float x = (uint32_t)(key >> 32) == kKeyNan ? __builtin_nanf("") : key_value((uint32_t)(key >> 32));
  a.top_indices[row * a.top + rank] = some ? (int64_t)(0xFFFFFFFFu - (uint32_t)key) : -1;
  a.top_logprobs[row * a.top + rank] = some ? (x - st.m) * a.r.scale - st.log_s : -kInf;
}

// One row, or one chunk of it, a group.  Bound by memory: 4096 x 49408 bf16 with 20 alternatives 84 us = 4.8 TB/s (78
// without alternatives, 107 with 100), 2048 x 131071 in two chunks a row 127 with the join = 4.2.  Rows that a
// wave holds are bound by its instructions, most of them the alternatives': 65536 x 1203 fp16, top 20, 62 us = 2.5 TB/s
// with the VALU busy for 0.87 of it; small calls by the launch (300 x 65 5.7 us, 1728 x 1203 with a mask 8.3, 1 x 49408 6.9).
// Rows off the common way: a mask for each row 150 us at 4096 x 49408, -inf among the logits 120, all equal 775, NaN in every
// row 1745.
template <typename T, int NT, int NV, bool MASK>
__global__ __launch_bounds__(kBlock<NT>, kWaves<NT>) void score_kernel(ScoreArgs a) {
  constexpr int G = kGroups<NT>, E = kPer<T>, CAP = kListCap<NT>;
  __shared__ __attribute__((aligned(16))) float part_max[NT == 64 ? 1 : kParts];
  __shared__ float tmp_s[NT / 64], tmp_t[NT / 64];
  constexpr int VECS = kVecCap<NT>;
  __shared__ u32x4_t vecs[G][VECS];
  __shared__ int vec_col[G][VECS], vecs_n[G];
  __shared__ uint64_t list[G][CAP];
  __shared__ int list_n[G], last_n[G];
  const int64_t index = group_index<NT>();
  if (index >= a.r.rows * a.sp.parts) return;
  const int64_t row = a.sp.parts == 1 ? index : index / a.sp.parts;
  const int part = (int)(index - row * a.sp.parts);
  const int g = NT == 64 ? threadIdx.x / 64 : 0, t = group_tid<NT>();
  const int64_t first = part * a.sp.chunk;
  const int64_t left = a.r.vocab - first;
  const T* x = static_cast<const T*>(a.r.x) + row * a.r.stride + first;
  const bool whole = a.sp.parts == 1;
  Given given;
  given.id = whole ? given_id(a, row, t) : -1;
  Tile<T, NT, NV> tile;
  tile.load(x, (int)(left < a.sp.chunk ? left : a.sp.chunk), a.r.big);
  given.x = given.id < 0 ? 0.f : given_logit<T>(a, row, given.id);
  if constexpr (MASK) tile.apply_mask(a.r.mask + row * a.r.mask_stride + first);
  if (t == 0) vecs_n[g] = list_n[g] = 0;

  // the largest logit, and a bound for the alternatives
  float vmax[NV], mine = tile.single, m, bound = kInf;
  tile.each([&](u32x4_t q, int vi) {
    vmax[vi] = vec_max<T>(q);
    mine = max3(mine, vmax[vi], vmax[vi]);
  });
  if constexpr (NT == 64) {
    m = wave64_max(mine);
    if (a.top) {
      // Parts: the lanes' own places, or the vectors, where there are twice as many as are wanted; else each place for itself
      // (exact, but eight times the counting.  Vectors / places, us: 16384 x 2000 bf16, 100 alternatives, 64 / 91; 8192 x 1203
      // fp16, 50 21 / 38, 100 - 1.5 vectors for each - 49 / 47, 128 86 / 54: too many keys to rank).  So few places that ranking
      // all of them takes less than that: no bound (19200 x 65 fp16, 5 alternatives 27 / 35, x 17 15 / 35; 121 places 50 / 36).
      if (tile.n <= 96 && tile.nvec < 2 * a.top) {
        bound = kLowest;
      } else if (a.top <= 32 && tile.nvec >= 2 * a.top) {
        bound = bound_by_bits(a.top, [&](float v) { return __popcll(__ballot(mine >= v)); });
      } else if (tile.nvec >= 2 * a.top) {
        bound = bound_by_bits(a.top, [&](float v) {
          int n = 0;
#pragma unroll
          for (int vi = 0; vi < NV; ++vi)
            if (vi < tile.nv) n += __popcll(__ballot(tile.has_vec(vi) && vmax[vi] >= v));
          return n;
        });
      } else {
        bound = bound_by_bits(a.top, [&](float v) {
          int n = __popcll(__ballot(tile.single >= v));
#pragma unroll
          for (int vi = 0; vi < NV; ++vi)
            if (vi < tile.nv) {
              const bool here = tile.has_vec(vi);
#pragma unroll
              for (int i = 0; i < E; ++i) n += __popcll(__ballot(here && elem<T>(tile.v[vi], i) >= v));
            }
          return n;
        });
      }
    }
  } else {
    constexpr int W = NT / kParts;  // threads of a part
    float p = mine;
    if constexpr (W >= 2) p = fmaxf(p, __shfl_xor(p, 1, 64));
    if constexpr (W >= 4) p = fmaxf(p, __shfl_xor(p, 2, 64));
    if (t % W == 0) part_max[t / W] = p;
    __syncthreads();
    const float4 q = *reinterpret_cast<const float4*>(&part_max[t % 64 * 4]);
    m = wave64_max(fmaxf(fmaxf(q.x, q.y), fmaxf(q.z, q.w)));
    if (a.top) {
      const float four = fmaxf(fmaxf(q.x, q.y), fmaxf(q.z, q.w));
      if (a.top <= 32) {
        bound = bound_by_count(-wave64_max(-four), m, a.top, [&](float v) { return __popcll(__ballot(four >= v)); });
      } else {
        const float least = -wave64_max(-fminf(fminf(q.x, q.y), fminf(q.z, q.w)));
        bound = bound_by_count(least, m, a.top, [&](float v) {
          return __popcll(__ballot(q.x >= v)) + __popcll(__ballot(q.y >= v)) + __popcll(__ballot(q.z >= v)) +
                 __popcll(__ballot(q.w >= v));
        });
      }
    }
  }

  // sums, and the places at or above the bound
  const Ref ref(m, a.r.scale * kLog2e);
  m = ref.m;
  tile.pack();
  Sums sums;
  const auto keep = [&](u32x4_t q, int col) {  // a vector that holds places at or above the bound
    const int at = atomicAdd(&vecs_n[g], 1);
    if (at < VECS) {
      vecs[g][at] = q;
      vec_col[g][at] = col;
    }
  };
  if constexpr (NT == 64) group_sync<NT>();  // (list_n is 0)
  tile.each([&](u32x4_t q, int vi) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float d = elem_fma<T>(q, i, ref.c, -ref.b);
      if constexpr (MASK) sums.add(d);
      else sums.add_finite(d);
    }
    if (vmax[vi] >= bound) keep(q, tile.vec_col(vi));
  });
  sums.add(__builtin_fmaf(tile.single, ref.c, -ref.b));
  if (tile.single >= bound) {
    const unsigned none = neg_inf_bits<T>();
    u32x4_t q = u32x4_t{none, none, none, none};
    if constexpr (sizeof(T) == 4) q[0] = __float_as_uint(tile.single);
    else q[0] = (none & 0xFFFF0000u) | __builtin_bit_cast(unsigned short, to16<T>(tile.single));
    keep(q, tile.single_col());
  }
  const auto reduce = [&]() {
    sums.s = wave64_sum(sums.s);
    sums.t = wave64_sum(sums.t);
    if constexpr (NT == 64) {
      group_sync<NT>();
    } else {
      if (t % 64 == 0) {
        tmp_s[t / 64] = sums.s;
        tmp_t[t / 64] = sums.t;
      }
      __syncthreads();
      sums.s = tmp_s[0];
      sums.t = tmp_t[0];
#pragma unroll
      for (int w = 1; w < NT / 64; ++w) {
        sums.s += tmp_s[w];
        sums.t += tmp_t[w];
      }
    }
  };
  reduce();
  if (!ref.fused || (sums.t != sums.t && sums.s == sums.s)) {
    // logits past what the fused form takes, or -inf among them: again, in the form that takes everything
    if constexpr (NT != 64) __syncthreads();
    sums = Sums();
    tile.pack();
    tile.each([&](u32x4_t q, int) {
#pragma unroll
      for (int i = 0; i < E; ++i) sums.add((elem<T>(q, i) - m) * ref.c);
    });
    sums.add((tile.single - m) * ref.c);
    reduce();
  } else {
    sums.relative_to_m(ref);
  }

  RowStats st;
  if (whole) {
    st = row_stats(m, sums.s, sums.t);
    if (t == 0) write_row(a, row, st);
    write_given<T>(a, row, st, t, NT, given);
  } else if (t == 0) {
    float* p = a.part_sums + index * 4;
    p[0] = m;
    p[1] = sums.s;
    p[2] = sums.t;
  }
  if (a.top == 0) return;
  const auto put = [&](int rank, uint64_t key) {
    if (whole) write_top(a, row, st, rank, key);
    else a.part_keys[index * a.top + rank] = key;
  };
  const int held = vecs_n[g];
  if (held <= VECS) {  // the places of those vectors, all threads at once
    const T* all = reinterpret_cast<const T*>(vecs[g]);
    for (int i = t; i < held * E; i += NT) {
      const float v = (float)all[i];
      if (v >= bound) {
        const int at = atomicAdd(&list_n[g], 1);
        if (at < CAP) list[g][at] = place_key(v, (uint32_t)(first + vec_col[g][i / E] + i % E));
      }
    }
  }
  group_sync<NT>();
  int n = list_n[g];
  if (held > VECS || n > CAP || sums.s != sums.s) {
    // Too many equal values at the bound, or NaN: the top-th key itself, by halving over the row, then the last place that
    // holds an equal one and still counts.  (From memory: the tile's registers are not held for the rare case.)
    const uint8_t* mask = MASK ? a.r.mask + row * a.r.mask_stride + first : nullptr;
    const auto key_at = [&](int j) { return order_key(MASK && !mask[j] ? -kInf : (float)x[j]); };
    const auto count = [&](int places, auto yes) {
      int c = 0;
#pragma unroll 8
      for (int j = t; j < places; j += NT) c += yes(key_at(j));
      float sum = wave64_sum((float)c);  // (a chunk has less than 2^24 places)
      if constexpr (NT != 64) {
        if (t % 64 == 0) tmp_s[t / 64] = sum;
        __syncthreads();
        sum = 0.f;
        for (int w = 0; w < NT / 64; ++w) sum += tmp_s[w];
        __syncthreads();
      }
      return (int)sum;
    };
    // keys of one value: those of [v, v + unit)
    constexpr uint32_t unit = sizeof(T) == 4 ? 1u : __is_same(T, f16_t) ? 1u << 13 : 1u << 16;
    uint32_t lo = kKeyNegInf + 1, hi = kKeyNan & ~(unit - 1);
    int above = 0;                       // places with a key of `hi` or more: fewer than top
    if (sums.s == sums.s) {              // (the bound is right: top places reach it, or it is the lowest number)
      lo = order_key(bound) & ~(unit - 1);
      hi = (order_key(m) & ~(unit - 1)) + unit;
    } else {
      above = count(tile.n, [&](uint32_t k) { return k >= hi; });
      if (above >= a.top) lo = hi, above = 0;
    }
    while (lo < hi && hi - lo > unit) {
      const uint32_t mid = lo + (hi - lo) / 2 / unit * unit;
      const int c = count(tile.n, [&](uint32_t k) { return k >= mid; });
      if (c >= a.top) lo = mid;
      else hi = mid, above = c;
    }
    // the waves look through a stretch of the row each for places of the value `lo`; the wave in whose stretch enough of
    // them come together looks for that place
    const auto equal = [&](int j) {
      const uint32_t k = j < tile.n ? key_at(j) : 0;
      return k > kKeyNegInf && k >= lo && k - lo < unit;
    };
    const int wave = NT == 64 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = t % 64;
    const int stretch = (tile.n + NT - 1) / NT * 64, begin = wave * stretch, need = a.top - above;
    int mine = 0, before = 0;
#pragma unroll 8
    for (int j = begin + lane; j < begin + stretch; j += 64) mine += equal(j);
    mine = (int)wave64_sum((float)mine);
    if (t == 0) last_n[g] = tile.n - 1;
    if constexpr (NT != 64) {
      if (lane == 0) tmp_s[wave] = (float)mine;
      __syncthreads();
      for (int w = 0; w < wave; ++w) before += (int)tmp_s[w];
    }
    if (before < need && before + mine >= need) {
      for (int j = begin; before < need; j += 64) {
        const uint64_t lanes = __ballot(equal(j + lane));
        const int c = __popcll(lanes);
        if (before + c >= need) {  // the (need - before)-th of these lanes
          const int at = __builtin_amdgcn_mbcnt_hi((unsigned)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)lanes, 0));
          if ((lanes >> lane & 1) && before + at + 1 == need) last_n[g] = j + lane;
        }
        before += c;
      }
    }
    group_sync<NT>();
    const int last = last_n[g];  // places of value `lo` up to here count
    if (t == 0) list_n[g] = 0;
    group_sync<NT>();
    for (int j = t; j < tile.n; j += NT) {
      const uint32_t k = key_at(j);
      if (k <= kKeyNegInf || k < lo || (k - lo < unit && j > last)) continue;
      const int at = atomicAdd(&list_n[g], 1);
      if (at < CAP) list[g][at] = (uint64_t)k << 32 | (0xFFFFFFFFu - (uint32_t)(first + j));
    }
    group_sync<NT>();
    n = list_n[g] < CAP ? list_n[g] : CAP;
  }
  constexpr int R = NT == 64 ? 2 : 8;  // lanes that count for one key
  for (int i = t / R; i < n; i += NT / R) {
    const uint64_t key = list[g][i];
    int rank = 0;
#pragma unroll 8
    for (int k = t % R; k < n; k += R) rank += list[g][k] > key;
    rank = R == 8 ? sum8(rank) : sum2(rank);
    if (t % R == 0 && rank < a.top) put(rank, key);
  }
  for (int i = n + t; i < a.top; i += NT) put(i, 0);
}

// The chunks of a row joined: sums brought to the largest m, in the chunks' order, and the chunks' lists.  Of every list its
// ceil(top / chunks)-th key: at least `top` keys reach the least of these, and each of those is ranked by the number of larger
// ones.  Where they are too many for the LDS (equal values in most lists), a key's rank is its place in its own list plus,
// for each other list, how many keys of that are larger (a binary search).  Bound by its chain of dependent steps: 16 rows of
// seven chunks with 100 alternatives 8.9 us, 2048 rows of two with 64 9.5.
constexpr int kJoinCap = 2048;
template <typename T>
__global__ __launch_bounds__(kThreads) void score_join_kernel(ScoreArgs a) {
  __shared__ uint64_t list[kJoinCap];
  __shared__ int list_n;
  const int64_t row = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  if (row >= a.r.rows) return;
  const int t = threadIdx.x, parts = a.sp.parts, top = a.top;
  const float* p = a.part_sums + row * parts * 4;
  const float c = a.r.scale * kLog2e;
  Given given;
  given.id = given_id(a, row, t);
  given.x = given.id < 0 ? 0.f : given_logit<T>(a, row, given.id);
  // every wave for itself: no exchange
  float m = -kInf, s = 0.f, u = 0.f;
  for (int i = t % 64; i < parts; i += 64)
    if (p[i * 4 + 1] != 0.f) m = fmaxf(m, p[i * 4]);
  m = wave64_max(m);
  if (m == -kInf) m = 0.f;
  for (int i = t % 64; i < parts; i += 64) {
    const float si = p[i * 4 + 1], ui = p[i * 4 + 2];
    if (si == 0.f) continue;
    const float d = (p[i * 4] - m) * c, f = __builtin_amdgcn_exp2f(d);
    s += f * si;
    u += f * (ui + si * fmaxf(d, -200.f));
  }
  s = wave64_sum(s);
  u = wave64_sum(u);
  const RowStats st = row_stats(m, s, u);
  if (t == 0) write_row(a, row, st);
  write_given<T>(a, row, st, t, kThreads, given);
  if (top == 0) return;

  const int64_t total = (int64_t)parts * top;
  const uint64_t* all = a.part_keys + row * total;
  const int share = (top + parts - 1) / parts - 1;
  if (t == 0) list_n = 0;
  uint64_t bound = ~0ull;  // (by every wave for itself; 0: a list has fewer keys, and all of them are looked at)
  for (int p = t % 64; p < parts; p += 64) {
    const uint64_t k = all[(int64_t)p * top + share];
    bound = k < bound ? k : bound;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t k = __shfl_xor(bound, o, 64);
    bound = k < bound ? k : bound;
  }
  if (bound == 0) bound = 1;
  __syncthreads();
  for (int64_t i = t; i < total; i += kThreads) {
    const uint64_t key = all[i];
    if (key < bound) continue;
    const int at = atomicAdd(&list_n, 1);
    if (at < kJoinCap) list[at] = key;
  }
  __syncthreads();
  const int n = list_n;
  if (n <= kJoinCap) {
    for (int i = t / 8; i < n; i += kThreads / 8) {  // eight lanes count for one key
      const uint64_t key = list[i];
      int rank = 0;
#pragma unroll 8
      for (int k = t % 8; k < n; k += 8) rank += list[k] > key;
      rank = sum8(rank);
      if (t % 8 == 0 && rank < top) write_top(a, row, st, rank, key);
    }
  } else {
    for (int64_t i = t; i < total; i += kThreads) {
      const uint64_t key = all[i];
      if (key < bound) continue;
      const int own = (int)(i / top);
      int64_t rank = i - (int64_t)own * top;
      for (int p = 0; p < parts && rank < top; ++p) {
        if (p == own) continue;
        const uint64_t* other = all + (int64_t)p * top;
        int lo = 0;  // keys of the other list before `lo` are larger
        for (int step = kMaxTop; step > 0; step /= 2) {
          const int at = lo + step < top ? lo + step : top;
          lo = other[at - 1] > key ? at : lo;
        }
        rank += lo;
      }
      if (rank < top) write_top(a, row, st, (int)rank, key);
    }
  }
  for (int i = n + t; i < top; i += kThreads) write_top(a, row, st, i, 0);
}

// ---- the teacher's list of one row ----------------------------------------------------------------------------
struct TeacherArgs {
  const void* ids;
  const float* v;
  int wide_ids, n, tail;
};
// one entry: its place (-1: absent, or no place of the vocabulary) and its log probability (-inf: absent; NaN: loud)
__device__ __forceinline__ float teacher_entry(const TeacherArgs& a, int64_t row, int64_t vocab, int i, int& id) {
  const int64_t j = load_id(a.ids, a.wide_ids, row * a.n + i);
  float v = a.v[row * a.n + i];
  if (j < 0) v = -kInf;
  if (j >= vocab && v != -kInf) v = __builtin_nanf("");
  id = v == -kInf || j >= vocab ? -1 : (int)j;
  return v;
}
// q = e^(v - log_norm): the softmax of the row's entries, or (tail) e^v as they are and a bucket for what is left of 1,
// a difference from 1 that is taken in 64 bits
struct Teacher {
  double log_norm, q_rest;
  float q_sum;
  bool some;  // there is an entry at all
};
template <int CAP>
struct TeacherList {  // in LDS
  int id[CAP];
  float v[CAP], x[CAP];  // x: the student's logit there
  Teacher t;
};
// e^v in 64 bits for what stands in a list: v = n log 2 + r, the series of e^r (|r| <= 0.35: the 12th term is below 1e-14).
// (The library's exp is what would set the kernel's registers.)
__device__ __forceinline__ double exp64(double v) {
  const double n = __builtin_rint(v * 1.4426950408889634), r = __builtin_fma(n, -0.69314718055994531, v);
  double p = 1.0;
#pragma unroll
  for (int k = 11; k > 0; --k) p = __builtin_fma(p * (1.0 / k), r, 1.0);
  return v < -200.0 ? 0.0 : __builtin_ldexp(p, (int)n);
}
// log s in 64 bits: that of s in fp32, and one step of Newton's on e^y = s (which squares its error of 2^-24).  log 1 = 0: the
// part that the exponent leaves lies around 1.
__device__ __forceinline__ double log64(double s) {
  if (s == 0) return -__builtin_inf();
  int n = __builtin_amdgcn_frexp_exp(s);
  double part = __builtin_ldexp(s, -n);
  if (part < 0.70710678) part += part, n -= 1;
  const double y = logf((float)part);
  return y + (part * exp64(-y) - 1.0) + n * 0.69314718055994531;
}
// By one wave (every lane of it), for the group.  `id`, `v`: the lane's first entry (teacher_entry), fetched before the row
// was; x (or nullptr): the student's row, whose listed logits are fetched too.
template <typename T, int CAP>
__device__ __forceinline__ void teacher_row(const TeacherArgs& a, int64_t row, int64_t vocab, const T* x, int id, float v,
                                            TeacherList<CAP>& s) {
  const int lane = threadIdx.x % 64;
  float best = -kInf, some = 0.f;
  for (int i = lane; i < a.n; i += 64) {
    if (i != lane) v = teacher_entry(a, row, vocab, i, id);
    s.id[i] = id;
    s.v[i] = v;
    if (x) s.x[i] = id < 0 ? -kInf : (float)x[id];
    best = fmaxf(best, v);
    if (v != -kInf) some = 1.f;
  }
  best = wave64_max(best);
  some = wave64_max(some);
  if (a.tail || best == -kInf) best = 0.f;  // (no entry: every q is 0)
  group_sync<64>();
  double sum = 0;
  for (int i = lane; i < a.n; i += 64) sum += exp64((double)s.v[i] - best);
  sum = wave64_sum(sum);
  const double log_norm = a.tail || sum == 0 ? best : best + log64(sum);
  float q_sum = 0.f;
  for (int i = lane; i < a.n; i += 64) q_sum += expf((float)(s.v[i] - log_norm));
  q_sum = wave64_sum(q_sum);
  if (lane == 0) s.t = {log_norm, a.tail && !(sum > 1) ? 1 - sum : 0, q_sum, some != 0.f};
}

// ---- distill_top_logits -----------------------------------------------------------------------------------------
struct DistillArgs {
  Rows r;
  Split sp;
  TeacherArgs t;
  float *loss, *stats;
  float* part_sums;  // [rows, parts, 2]: m, S of a chunk (tail: of its places outside the list)
};
// What the backward pass needs of a row: m, 1 / S (0: the student has nothing); the same outside the list; the student's
// probability there; the teacher's log_norm, q_sum (-1: no entry) and, with the tail, bucket - without (log_norm is 0 with it),
// what log_norm's rounding left: a list may stand at any height, and 2^-24 of it would be a factor of all its q
constexpr int kStats = 8;
// Rows of so many are summed in 64 bits, whoever works on them (few classes: a loss of 1e-4 and less is ordinary).  fp32 /
// 64 bits, us: 300 x 65 fp32 5.6 / 6.0, 19200 x 65 fp32 21 / 26, fp16 (eight places a lane) 21 / 30, x 128 fp16 20 / 30.  A
// detector's 65 classes are well inside; longer rows keep what their fp32 sum leaves in log S.
constexpr int kExactPlaces = 128;
__device__ __forceinline__ void write_no_teacher(const DistillArgs& a, int64_t row) {
  a.loss[row] = 0.f;
  a.stats[row * kStats + 6] = -1.f;
}

// The end of a row, by one group: `m` and `s` are the row's largest logit and sum (tail: of the places outside the list;
// the listed ones are added here, each place once).  Where teacher and student nearly agree the loss is a difference of equal
// logarithms: those, the list's sums and (short rows) all sums are taken in 64 bits.  EXACT: so are the terms and their sum
// (weights and the bucket in fp32 leave the loss off by 2^-24 of the terms, 2e-5 of a loss of 1e-4; 300 x 65 5.3 us without,
// 5.6 with); not in long rows, whose fp32 sum leaves more than that in log S (4096 x 49408 91 / 95).
template <int NT, bool EXACT, int CAP>
__device__ __forceinline__ void finish_distill(const DistillArgs& a, int64_t row, const TeacherList<CAP>& te, bool distinct,
                                               float m, double s,
                                               std::conditional_t<EXACT, double, float>* tmp) {
  using F = std::conditional_t<EXACT, double, float>;
  const int t = group_tid<NT>(), n = a.t.n;
  const float scale = a.r.scale, mo = m;
  const double so = s;
  float p_o = 1.f;
  if (a.t.tail) {
    float peak = so == 0 ? -kInf : mo;
    // (few values: every wave looks at all of them)
    for (int i = t % 64; i < n; i += 64)
      peak = fmaxf(peak, te.x[i]);
    peak = wave64_max(peak);
    m = peak == -kInf ? 0.f : peak;
    s = 0;
    for (int i = t % 64; i < n; i += 64) {
      bool first = te.id[i] >= 0;
      if (!distinct)
        for (int k = 0; k < i; ++k) first = first && te.id[k] != te.id[i];
      if (first) s += exp64(((double)te.x[i] - m) * scale);
    }
    s = wave64_sum(s);
    const double outside = so == 0 ? 0 : so * exp64(((double)mo - m) * scale);
    s += outside;
    p_o = (float)(outside / s);
  }
  const double log_s = log64(s);
  F loss = 0;
  for (int i = t; i < n; i += NT) {
    const double v = te.v[i], log_q = v - te.t.log_norm;
    F q;
    if constexpr (EXACT) q = exp64(log_q);
    else q = expf((float)log_q);
    if ((float)q == 0.f) continue;
    const double y = te.id[i] < 0 ? v : te.x[i];  // (an id that the vocabulary does not have: v is NaN)
    loss += q * (y == -kInf && s == s ? (F)kInf : (F)(log_q - (y - m) * scale + log_s));
  }
  loss = group_sum<NT>(loss, tmp);
  if (t == 0) {
    const double q_rest = !a.t.tail || so == 0 ? 0 : te.t.q_rest;
    if (q_rest != 0) loss += (F)q_rest * (F)(log64(q_rest) - ((double)mo - m) * scale - log64(so) + log_s);
    const float rest = (float)q_rest;
    a.loss[row] = (float)loss;
    float* st = a.stats + row * kStats;
    st[0] = m;
    st[1] = s == 0 ? 0.f : (float)(1 / s);
    st[2] = mo;
    st[3] = so == 0 ? 0.f : (float)(1 / so);
    st[4] = p_o;
    const float norm = (float)te.t.log_norm;
    st[5] = norm;
    st[6] = te.t.q_sum;
    st[7] = a.t.tail ? rest : (float)(te.t.log_norm - norm);
  }
}

// One row, or one chunk of it, a group; the teacher's list is read beside the row by the group's first wave.  TAIL: the sum
// over the places outside the list is what is kept (1 - sum of the listed p would lose it to rounding), the listed places
// being known by the bits of a map in LDS: vectors first (a vector's bits are a byte, or half of one), then the single ones.
// Bound by memory: 4096 x 49408 bf16, 64 entries, 83 us = 4.9 TB/s; 1024 x 100003 fp32 with the bucket, in four chunks a row,
// 69 + 10.2 for the join = 5.1; 2400 x 1203 fp16 with the bucket 10.8, 300 x 65 6.4: there the list's exponentials and logarithms
// in 64 bits, one after the other.
template <typename T, int NT, int NV, bool TAIL, int LIST>
__global__ __launch_bounds__(kBlock<NT>, kWaves<NT>) void distill_kernel(DistillArgs a) {
  constexpr int G = kGroups<NT>, E = kPer<T>, WORDS = TAIL ? NT * NV * E / 32 + 1 : 1;
  __shared__ TeacherList<LIST> te[G];
  __shared__ unsigned map[G][WORDS];
  __shared__ int twice[G];
  __shared__ float tmp_m[NT / 64], tmp_s[NT / 64];
  constexpr bool EXACT = NT <= 256;  // (workgroups of 512 have longer rows)
  __shared__ double tmp_d[NT / 64];
  __shared__ std::conditional_t<EXACT, double, float> tmp_l[NT / 64];
  const int64_t index = group_index<NT>();
  if (index >= a.r.rows * a.sp.parts) return;
  const int64_t row = a.sp.parts == 1 ? index : index / a.sp.parts;
  const int part = (int)(index - row * a.sp.parts);
  const int g = NT == 64 ? threadIdx.x / 64 : 0, t = group_tid<NT>();
  const int64_t first = part * a.sp.chunk;
  const int64_t left = a.r.vocab - first;
  const T* x = static_cast<const T*>(a.r.x) + row * a.r.stride + first;
  const bool whole = a.sp.parts == 1;
  int id = -1;
  float v = 0.f;
  if ((TAIL || whole) && t < 64 && t < a.t.n) v = teacher_entry(a.t, row, a.r.vocab, t, id);
  Tile<T, NT, NV> tile;
  tile.load(x, (int)(left < a.sp.chunk ? left : a.sp.chunk), a.r.big);
  if (t == 0) twice[g] = 0;
  if constexpr (TAIL) {
    for (int i = t; i < WORDS; i += NT) map[g][i] = 0;
    group_sync<NT>();
  }
  if ((TAIL || whole) && t < 64) {
    teacher_row(a.t, row, a.r.vocab, whole ? x : nullptr, id, v, te[g]);
    if constexpr (TAIL) {
      for (int i = t; i < a.t.n; i += 64) {
        const int64_t col = te[g].id[i] - first;
        if (te[g].id[i] < 0 || col < 0 || col >= tile.n) continue;
        const int nv = tile.nvec * E, bit = col < nv ? (int)col : NT * NV * E + (int)col - nv;
        if (atomicOr(&map[g][bit / 32], 1u << bit % 32) >> bit % 32 & 1) twice[g] = 1;
      }
    }
  }
  // (TAIL: the largest of all places, listed or not - the map is not there yet)
  const auto largest = [&]() {
    float m = wave64_max(tile.max());
    if constexpr (NT != 64) {
      if (t % 64 == 0) tmp_m[t / 64] = m;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NT / 64; ++w) m = fmaxf(m, tmp_m[w]);
    } else {
      group_sync<NT>();
    }
    return m;
  };
  float m = largest();
  if ((TAIL || whole) && !te[g].t.some) {  // no teacher: no loss
    if (t == 0 && whole) write_no_teacher(a, row);
    return;
  }
  if constexpr (TAIL) {  // what the list holds is left out
    unsigned bits[NV];
#pragma unroll
    for (int vi = 0; vi < NV; ++vi)  // (the map covers all NV: one wait for all of them)
      bits[vi] = map[g][(vi * NT + t) * E / 32] >> (vi * NT + t) * E % 32 & ((1u << E) - 1);
#pragma unroll
    for (int vi = 0; vi < NV; ++vi)
      if (vi < tile.nv && __any(bits[vi] != 0)) {
#pragma unroll
        for (int i = 0; i < E; ++i) drop<T>(tile.v[vi], i, bits[vi] >> i & 1);
      }
    if (t < 32 && map[g][NT * NV * E / 32] >> t & 1) tile.single = -kInf;
  }
  const auto sum = [&]() -> double {
    const Ref ref(m, a.r.scale * kLog2e);
    m = ref.m;
    tile.pack();
    if constexpr (EXACT) {
      if (whole && tile.n <= kExactPlaces) {
        const auto e = [&](float v) { return exp64(((double)v - m) * a.r.scale); };
        double s = e(tile.single);
        if (tile.has_vec(0)) {  // (nobody has more than one)
#pragma unroll
          for (int i = 0; i < E; ++i) s += e(elem<T>(tile.v[0], i));
        }
        return group_sum<NT>(s, tmp_d);
      }
    }
    float s = 0.f;
    if (ref.fused) {
      tile.each([&](u32x4_t q, int) {
#pragma unroll
        for (int i = 0; i < E; ++i) s += __builtin_amdgcn_exp2f(elem_fma<T>(q, i, ref.c, -ref.b));
      });
      s += __builtin_amdgcn_exp2f(__builtin_fmaf(tile.single, ref.c, -ref.b));
    } else {
      tile.each([&](u32x4_t q, int) {
#pragma unroll
        for (int i = 0; i < E; ++i) s += __builtin_amdgcn_exp2f((elem<T>(q, i) - m) * ref.c);
      });
      s += __builtin_amdgcn_exp2f((tile.single - m) * ref.c);
    }
    return group_sum<NT>(s, tmp_s) / ref.one;
  };
  double s = sum();
  if (TAIL && s < 1e-30) {  // the largest is a listed one, far above all others: again, from the largest of those
    if constexpr (NT != 64) __syncthreads();
    m = largest();
    s = sum();
  }
  if (whole) {
    finish_distill<NT, EXACT>(a, row, te[g], TAIL && !twice[g], m, s, tmp_l);
  } else if (t == 0) {
    a.part_sums[index * 2] = m;
    a.part_sums[index * 2 + 1] = (float)s;
  }
}

// The chunks of a row joined, as above: of the sums, and the loss from the list (whose logits are read here).  Places listed
// twice are looked for by comparing each entry with those before it: nothing for 32 entries, most of the time for many
// (1024 x 100003 fp32 with the bucket, forward: 32 entries 82 us, 128 103, 512 308, 1024 805).
template <typename T>
__global__ __launch_bounds__(kThreads) void distill_join_kernel(DistillArgs a) {
  __shared__ TeacherList<kMaxList> te;
  __shared__ float tmp[kThreads / 64];
  const int64_t row = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  if (row >= a.r.rows) return;
  const int t = threadIdx.x, parts = a.sp.parts;
  if (t < 64) {
    int id = -1;
    const float v = t < a.t.n ? teacher_entry(a.t, row, a.r.vocab, t, id) : 0.f;
    teacher_row(a.t, row, a.r.vocab, static_cast<const T*>(a.r.x) + row * a.r.stride, id, v, te);
  }
  __syncthreads();
  if (!te.t.some) {
    if (t == 0) write_no_teacher(a, row);
    return;
  }
  const float* p = a.part_sums + row * parts * 2;
  float m = -kInf, s = 0.f;
  for (int i = t % 64; i < parts; i += 64)
    if (p[i * 2 + 1] != 0.f) m = fmaxf(m, p[i * 2]);
  m = wave64_max(m);
  if (m == -kInf) m = 0.f;
  for (int i = t % 64; i < parts; i += 64)
    if (p[i * 2 + 1] != 0.f) s += p[i * 2 + 1] * __builtin_amdgcn_exp2f((p[i * 2] - m) * (a.r.scale * kLog2e));
  s = wave64_sum(s);
  finish_distill<kThreads, false>(a, row, te, false, m, s, tmp);
}

// ---- gradients --------------------------------------------------------------------------------------------------
// Both operators' gradients are, over the whole row, p'_j * (a0 + a1 * (log p_j + H)) with p' = e^(d' - log S'), and at
// the few listed places j (given tokens and alternatives; the teacher's list) b0 * p_j + ... plus the weights of the
// entries that name j.  A chunk is written whole first, then its listed places again, each by the first entry that names
// it with the weights of all of them, so that no sum depends on an order.
template <typename T, int NT, int NV, typename F>
__device__ __forceinline__ void write_dense(const Tile<T, NT, NV>& tile, T* g, bool past_cache, F value) {
#pragma unroll
  for (int vi = 0; vi < NV; ++vi)
    if (vi < tile.nv && tile.has_vec(vi)) {
      u32x4_t out;
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = __float_as_uint(value(elem<T>(tile.v[vi], i)));
      } else {
        typename T16<T>::vec8 o;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = to16<T>(value(elem<T>(tile.v[vi], i)));
        out = __builtin_bit_cast(u32x4_t, o);
      }
      u32x4_any* to = reinterpret_cast<u32x4_any*>(g + tile.vec_col(vi));
      if (past_cache) store16_policy<2>(g + tile.vec_col(vi), out);  // (nt; any alignment)
      else *to = out;
    }
  if (tile.has_single()) g[tile.single_col()] = to16<T>(value(tile.single));
}
// the listed places of a chunk; value(x, weight).  Each looks through the whole list (1024 x 100003 fp32: 32 entries 146 us, 1024
// 3106).
template <typename T, int NT, typename F>
__device__ __forceinline__ void write_listed(const int* id, const float* w, int n, const T* x, T* g, int64_t first, int count,
                                             F value) {
  for (int i = group_tid<NT>(); i < n; i += NT) {
    const int j = id[i];
    if (j < first || j >= first + count) continue;  // (-1: no place)
    float sum = 0.f;
    bool before = false;
    for (int k = 0; k < n; ++k)
      if (id[k] == j) {
        before = before || k < i;
        sum += w[k];
      }
    if (!before) g[j - first] = to16<T>(value((float)x[j - first], sum));
  }
}

struct ScoreGradArgs {
  Rows r;
  Split sp;
  const void* targets;
  int wide_ids, n_targets, top;
  const int64_t* top_indices;
  const float *stats, *g_logprobs, *g_lse, *g_entropy, *g_top;
  void* grad;
  int64_t grad_stride;
  bool write_past;       // the gradient goes past the cache
};

// One row a wave, or a chunk of 256 threads with four vectors each: what it needs beside the logits is in the forward pass's
// stats, so chunks need no join, and short ones keep more of them in flight.  Bound by memory: 2048 x 49408 fp16 67 us =
// 6.0 TB/s read and written (the forward pass has left part of the logits in the Infinity Cache), 777 x 1203 fp32 6.4 us.
template <typename T, int NT, int NV, bool MASK, int LIST>
__global__ __launch_bounds__(kBlock<NT>, kWaves<NT>) void score_grad_kernel(ScoreGradArgs a) {
  constexpr int G = kGroups<NT>;
  __shared__ int ids[G][LIST];
  __shared__ float ws[G][LIST];
  __shared__ float tmp[NT / 64];
  const int64_t index = group_index<NT>();
  if (index >= a.r.rows * a.sp.parts) return;
  const int64_t row = a.sp.parts == 1 ? index : index / a.sp.parts;
  const int64_t first = (index - row * a.sp.parts) * a.sp.chunk;
  const int64_t left = a.r.vocab - first;
  const T* xr = static_cast<const T*>(a.r.x) + row * a.r.stride;
  const uint8_t* mask = MASK ? a.r.mask + row * a.r.mask_stride : nullptr;
  T* g = static_cast<T*>(a.grad) + row * a.grad_stride + first;
  Tile<T, NT, NV> tile;
  tile.load(xr + first, (int)(left < a.sp.chunk ? left : a.sp.chunk), a.r.big);
  if constexpr (MASK) tile.apply_mask(mask + first);
  int* id = ids[NT == 64 ? threadIdx.x / 64 : 0];
  float* w = ws[NT == 64 ? threadIdx.x / 64 : 0];
  const float m = a.stats[row * 4], log_s = a.stats[row * 4 + 1], h = a.stats[row * 4 + 2], inv_s = a.stats[row * 4 + 3];
  const float scale = a.r.scale;
  const int nt = a.g_logprobs ? a.n_targets : 0, n = nt + (a.g_top ? a.top : 0);
  float sum = 0.f;
  for (int i = group_tid<NT>(); i < n; i += NT) {
    const int64_t j = i < nt ? load_id(a.targets, a.wide_ids, row * a.n_targets + i) : a.top_indices[row * a.top + i - nt];
    float v = i < nt ? a.g_logprobs[row * a.n_targets + i] : a.g_top[row * a.top + i - nt];
    if (j < 0) v = 0.f;                                                    // padding
    else if (j >= a.r.vocab) v = __builtin_nanf("");                      // (its log probability is NaN)
    else if ((MASK && !mask[j]) || (float)xr[j] == -kInf) v = 0.f;        // -inf whatever the logits: a constant
    id[i] = j < 0 || j >= a.r.vocab || v == 0.f ? -1 : (int)j;
    w[i] = v;
    sum += v;
  }
  sum = n ? group_sum<NT>(sum, tmp) : 0.f;  // (its barrier is the lists' too)
  if constexpr (NT == 64) group_sync<NT>();
  const float gh = a.g_entropy ? a.g_entropy[row] : 0.f;
  const float a0 = (a.g_lse ? a.g_lse[row] : 0.f) - sum;
  const bool empty = log_s == -kInf;
  // p_j (a0 - g_H (log p_j + H)) with p_j = e^d_j / S (not e^(d_j - log S): log S has lost digits to its size)
  const float c = scale * kLog2e, b0 = a0 - gh * (h - log_s), b1 = gh * kLn2;
  const auto dense = [&](float x) {
    const float d = (x - m) * c;
    return __builtin_amdgcn_exp2f(d) * inv_s * (b0 - b1 * fmaxf(d, -200.f));
  };
  if (empty) {
    write_dense<T, NT, NV>(tile, g, a.write_past, [](float) { return 0.f; });
    return;
  }
  write_dense<T, NT, NV>(tile, g, a.write_past, [&](float x) {
    const float v = dense(x) * scale;
    return MASK && x == -kInf ? 0.f : v;
  });
  if (n == 0) return;
  group_sync<NT>();
  write_listed<T, NT>(id, w, n, xr + first, g, first, tile.n, [&](float x, float v) { return (dense(x) + v) * scale; });
}

struct DistillGradArgs {
  Rows r;
  Split sp;
  TeacherArgs t;
  const float *stats, *g_loss;
  void* grad;
  int64_t grad_stride;
  bool write_past;       // the gradient goes past the cache
};

// As above.  4096 x 49408 bf16 151 us = 5.4 TB/s, 1024 x 100003 fp32 144 = 5.7, 2400 x 1203 fp16 7.1, 300 x 65 4.4.
template <typename T, int NT, int NV, int LIST>
__global__ __launch_bounds__(kBlock<NT>, kWaves<NT>) void distill_grad_kernel(DistillGradArgs a) {
  constexpr int G = kGroups<NT>;
  __shared__ int ids[G][LIST];
  __shared__ float ws[G][LIST];
  const int64_t index = group_index<NT>();
  if (index >= a.r.rows * a.sp.parts) return;
  const int64_t row = a.sp.parts == 1 ? index : index / a.sp.parts;
  const int64_t first = (index - row * a.sp.parts) * a.sp.chunk;
  const int64_t left = a.r.vocab - first;
  const T* x = static_cast<const T*>(a.r.x) + row * a.r.stride + first;
  T* g = static_cast<T*>(a.grad) + row * a.grad_stride + first;
  Tile<T, NT, NV> tile;
  tile.load(x, (int)(left < a.sp.chunk ? left : a.sp.chunk), a.r.big);
  int* id = ids[NT == 64 ? threadIdx.x / 64 : 0];
  float* w = ws[NT == 64 ? threadIdx.x / 64 : 0];
  const float* st = a.stats + row * kStats;
  const float m = st[0], inv_s = st[1], mo = st[2], inv_so = st[3], p_o = st[4], log_norm = st[5], q_sum = st[6];
  const float rest = a.t.tail ? st[7] : 0.f, norm_rest = a.t.tail ? 0.f : st[7];
  if (q_sum == -1.f || inv_s == 0.f) {
    write_dense<T, NT, NV>(tile, g, a.write_past, [](float) { return 0.f; });
    return;
  }
  for (int i = group_tid<NT>(); i < a.t.n; i += NT) {
    int j;
    w[i] = expf(teacher_entry(a.t, row, a.r.vocab, i, j) - log_norm - norm_rest);
    id[i] = j;
  }
  const float up = a.g_loss[row] * a.r.scale, c = a.r.scale * kLog2e;
  const bool tail = a.t.tail && inv_so != 0.f;
  const float q_all = q_sum + rest;
  // outside the list: p_j q_all - rest e^(z_j - lse_o) = e^(z_j - lse_o) (p_o q_all - rest), p_o the student's bucket
  const float from = tail ? mo : m, a0 = tail ? up * (p_o * q_all - rest) * inv_so : up * q_all * inv_s;
  write_dense<T, NT, NV>(tile, g, a.write_past, [&](float v) { return a0 * __builtin_amdgcn_exp2f((v - from) * c); });
  group_sync<NT>();
  write_listed<T, NT>(id, w, a.t.n, x, g, first, tile.n, [&](float v, float q) {
    return up * (__builtin_amdgcn_exp2f((v - m) * c) * inv_s * q_all - q);
  });
}

// ---- launches -----------------------------------------------------------------------------------------------------
// Who works on a row, by its length and its lists': a wave where its registers hold the row (four rows a workgroup, no
// barriers; by wave / 256 threads, us: 300 x 65 fp32, 5 alternatives 4.7 / 9.7, 16384 x 2000 fp16, 20 23 / 63, 65536 x 1203 62 / 233,
// its gradient 62 / 100), a workgroup of 256 threads with 8 vectors each, or of 512 with 16 (256 / 512: 2400 x 4500 bf16
// 11.9 / 26, 8192 x 16000 49 / 93) - beyond that the row is cut into equal chunks, which a second launch joins.  The chunks
// are as long as they can be, few rows or many: a quarter as long with 256 threads, the join has four times the lists (a
// quarter / whole, us with the join: 16 x 200003 fp32, 100 alternatives 23 / 19, 20 14.6 / 11.9, 1 x 262143 bf16 11.9 /
// 12.8, 32 x 131071 bf16 12.3 / 15.6).  Gradients need no join and take 256 threads with 4 vectors (2 or 8: within 5 %).
// Rows of 2049 .. 4096 places go to a wave with twice the vectors where there are few alternatives to look for (wave /
// workgroup, us: 32768 x 2500 bf16, 20 alternatives 54 / 96; 2400 x 2500 8.1 / 11.3; 8192 x 4000 fp32, 100 alternatives 61 / 52;
// 2000 x 3000 fp16, 20 entries and the bucket 9.7 / 15.2).  That few rows would take less in workgroups (1 x 3000 fp16 5.2 / 4.6,
// 300 x 4096 fp32 8.1 / 5.7, under calls that the host takes 17 us for) does not count: how many there are decides nothing, so
// that a row has the same bits in any batch.
constexpr int kBlockVecs = 8, kLongVecs = 16, kGradVecs = 4;
constexpr int kWaveList = 64;  // entries of a list that a wave's share of the LDS holds
struct Plan {
  int threads;  // 64, 256, 512
  bool twice;   // a wave with 2 * kWaveVecs vectors a lane
  Split sp;
};
int64_t capacity(int threads, int vecs, int dtype) { return (int64_t)threads * vecs * (dtype == OAKE_F32 ? 4 : 8); }
Split split(int64_t vocab, int64_t most) {  // equal chunks of at most `most` places, each but the last a multiple of 8
  const int64_t parts = (vocab + most - 1) / most, chunk = ((vocab + parts - 1) / parts + 7) / 8 * 8;
  return {chunk, (int)((vocab + chunk - 1) / chunk)};
}
Plan forward_plan(int64_t vocab, int dtype, int top, int list) {
  if (list <= kWaveList) {
    if (vocab <= kWavePlaces) return {64, false, {vocab, 1}};
    if (vocab <= 2 * kWavePlaces && top <= 32) return {64, true, {vocab, 1}};
  }
  if (vocab <= capacity(256, kBlockVecs, dtype)) return {256, false, {vocab, 1}};
  return {512, false, split(vocab, capacity(512, kLongVecs, dtype))};
}
Plan backward_plan(int64_t vocab, int dtype, int list) {
  if (vocab <= kWavePlaces && list <= kWaveList) return {64, false, {vocab, 1}};
  return {256, false, split(vocab, capacity(256, kGradVecs, dtype))};
}
dim3 grid_of(int64_t blocks) {
  const int64_t x = blocks < 1 << 20 ? blocks : 1 << 20;
  return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}
int64_t blocks_of(const Plan& p, int64_t rows) { return p.threads == 64 ? (rows + 3) / 4 : rows * p.sp.parts; }
dim3 grid_of(const Plan& p, int64_t rows) { return grid_of(blocks_of(p, rows)); }
constexpr int64_t kMostBlocks = (int64_t)65535 << 20;

// ---- host side ----------------------------------------------------------------------------------------------------
__attribute__((format(printf, 2, 3))) int refuse(int code, const char* fmt, ...) {
  char text[256];
  va_list ap;
  va_start(ap, fmt);
  std::vsnprintf(text, sizeof(text), fmt, ap);
  va_end(ap);
  return fail_without_handle(code, text);
}
// Logits that the 256 MB of Infinity Cache do not hold are read past it, and gradients of more than half of it written
// past it: lines that no one will find there are not written back in the next kernel's time.  us for a loss and its
// gradient, with / without: 4096 x 49408 bf16 236 / 255, 1024 x 100003 fp32 232 / 266; below, where the backward pass finds
// the logits in the cache, 62 / 60 (1024 x 49408 bf16) and 93 / 82 (32768 x 1203 fp16): not there.
bool past_cache(int64_t rows, int64_t vocab, int64_t bytes_each, int64_t limit) {
  return (double)rows * vocab * bytes_each > limit;
}
size_t element_size(int dtype) { return dtype == OAKE_F32 ? 4 : 2; }

int check_rows(const char* what, const void* x, int dtype, int64_t rows, int64_t vocab, int64_t stride, float scale) {
  if (dtype != OAKE_F32 && dtype != OAKE_F16 && dtype != OAKE_BF16)
    return refuse(OAKE_ERR_INVALID, "%s: the logits must be F32, F16 or BF16", what);
  if (rows < 0 || rows > INT32_MAX || vocab < 1 || vocab > INT32_MAX)
    return refuse(OAKE_ERR_INVALID, "%s: rows must be 0 .. 2^31 - 1 and vocab 1 .. 2^31 - 1", what);
  if (stride < 0) return refuse(OAKE_ERR_INVALID, "%s: a row stride is negative", what);
  if (!(scale > 0.f) || scale > 1e38f) return refuse(OAKE_ERR_INVALID, "%s: scale must be positive and at most 1e38", what);
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

template <typename T>
void run_score(const Plan& p, const ScoreArgs& a, hipStream_t s) {
  const dim3 grid = grid_of(p, a.r.rows);
#define OAKE_SCORE(NT, NV)                                                                    \
  if (a.r.mask) score_kernel<T, NT, NV, true><<<grid, kBlock<NT>, 0, s>>>(a);        \
  else score_kernel<T, NT, NV, false><<<grid, kBlock<NT>, 0, s>>>(a)
  if (p.twice) { OAKE_SCORE(64, 2 * kWaveVecs<T>); }
  else if (p.threads == 64) { OAKE_SCORE(64, kWaveVecs<T>); }
  else if (p.threads == 256) { OAKE_SCORE(256, kBlockVecs); }
  else { OAKE_SCORE(512, kLongVecs); }
#undef OAKE_SCORE
  if (a.sp.parts > 1) score_join_kernel<T><<<grid_of(a.r.rows), kThreads, 0, s>>>(a);
}
template <typename T>
void run_score_grad(const Plan& p, const ScoreGradArgs& a, hipStream_t s) {
  const dim3 grid = grid_of(p, a.r.rows);
  if (p.threads == 64) {
    if (a.r.mask) score_grad_kernel<T, 64, kWaveVecs<T>, true, kWaveList><<<grid, 256, 0, s>>>(a);
    else score_grad_kernel<T, 64, kWaveVecs<T>, false, kWaveList><<<grid, 256, 0, s>>>(a);
  } else {
    if (a.r.mask) score_grad_kernel<T, 256, kGradVecs, true, kMaxList + kMaxTop><<<grid, 256, 0, s>>>(a);
    else score_grad_kernel<T, 256, kGradVecs, false, kMaxList + kMaxTop><<<grid, 256, 0, s>>>(a);
  }
}
template <typename T>
void run_distill(const Plan& p, const DistillArgs& a, hipStream_t s) {
  const dim3 grid = grid_of(p, a.r.rows);
#define OAKE_DISTILL(NT, NV, LIST)                                                                  \
  if (a.t.tail) distill_kernel<T, NT, NV, true, LIST><<<grid, kBlock<NT>, 0, s>>>(a);      \
  else distill_kernel<T, NT, NV, false, LIST><<<grid, kBlock<NT>, 0, s>>>(a)
  if (p.twice) { OAKE_DISTILL(64, 2 * kWaveVecs<T>, kWaveList); }
  else if (p.threads == 64) { OAKE_DISTILL(64, kWaveVecs<T>, kWaveList); }
  else if (p.threads == 256) { OAKE_DISTILL(256, kBlockVecs, kMaxList); }
  else { OAKE_DISTILL(512, kLongVecs, kMaxList); }
#undef OAKE_DISTILL
  if (a.sp.parts > 1) distill_join_kernel<T><<<grid_of(a.r.rows), kThreads, 0, s>>>(a);
}
template <typename T>
void run_distill_grad(const Plan& p, const DistillGradArgs& a, hipStream_t s) {
  const dim3 grid = grid_of(p, a.r.rows);
  if (p.threads == 64) distill_grad_kernel<T, 64, kWaveVecs<T>, kWaveList><<<grid, 256, 0, s>>>(a);
  else distill_grad_kernel<T, 256, kGradVecs, kMaxList><<<grid, 256, 0, s>>>(a);
}
#define OAKE_BY_TYPE(dtype, run, ...)                       \
  do {                                                      \
    if ((dtype) == OAKE_F32) run<float>(__VA_ARGS__);       \
    else if ((dtype) == OAKE_F16) run<f16_t>(__VA_ARGS__);  \
    else run<bf16_t>(__VA_ARGS__);                          \
  } while (0)

// scratch of a forward call: [rows, parts, 4] fp32, then [rows, parts, top] keys
size_t scratch_bytes(int64_t rows, const Split& sp, int top) {
  return sp.parts == 1 ? 0 : (size_t)rows * sp.parts * (16 + 8 * (size_t)top);
}
int check_scratch(const char* what, const void* ws, size_t have, size_t need) {
  if (need == 0) return OAKE_OK;
  if (!ws || have < need) return refuse(OAKE_ERR_INVALID, "%s: the workspace has %zu of %zu bytes", what, ws ? have : 0, need);
  if ((uintptr_t)ws % 16) return refuse(OAKE_ERR_INVALID, "%s: the workspace is not 16-byte aligned", what);
  return OAKE_OK;
}

}  // namespace
}  // namespace oake

using namespace oake;

extern "C" {

int oake_logits_workspace(int64_t rows, int64_t vocab, int dtype, int top, size_t* bytes) {
  const char* what = "oake_logits_workspace";
  if (!bytes) return refuse(OAKE_ERR_INVALID, "%s: null pointer", what);
  if (int rc = check_rows(what, bytes, dtype, rows, vocab, vocab, 1.f)) return rc;
  if (top < 0 || top > kMaxTop) return refuse(OAKE_ERR_INVALID, "%s: top must be 0 .. %d", what, kMaxTop);
  *bytes = scratch_bytes(rows, forward_plan(vocab, dtype, top, 0).sp, top);
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
  const Plan p = forward_plan(vocab, dtype, top, 0);
  if (blocks_of(p, rows) > kMostBlocks) return refuse(OAKE_ERR_INVALID, "%s: too many rows of this length", what);
  if (int rc = check_scratch(what, d_workspace, workspace_bytes, scratch_bytes(rows, p.sp, top))) return rc;
  float* sums = static_cast<float*>(d_workspace);
  uint64_t* keys = p.sp.parts == 1 ? nullptr : reinterpret_cast<uint64_t*>(sums + rows * p.sp.parts * 4);
  const ScoreArgs a{{d_logits, rows, vocab, row_stride, d_mask, mask_stride, scale,
                     past_cache(rows, vocab, element_size(dtype), 256 << 20)}, p.sp,
                    d_targets, index_dtype == OAKE_I64, n_targets, top,
                    d_logprobs, d_lse, d_entropy, d_top_logprobs, d_stats, d_top_indices, sums, keys};
  OAKE_BY_TYPE(dtype, run_score, p, a, (hipStream_t)stream);
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
  const Plan p = backward_plan(vocab, dtype, (d_grad_logprobs ? n_targets : 0) + (d_grad_top ? top : 0));
  if (blocks_of(p, rows) > kMostBlocks) return refuse(OAKE_ERR_INVALID, "%s: too many rows of this length", what);
  const ScoreGradArgs a{{d_logits, rows, vocab, row_stride, d_mask, mask_stride, scale,
                         past_cache(rows, vocab, element_size(dtype), 256 << 20)}, p.sp,
                        d_targets, index_dtype == OAKE_I64, n_targets, top, d_top_indices,
                        d_stats, d_grad_logprobs, d_grad_lse, d_grad_entropy, d_grad_top, d_grad, grad_stride,
                        past_cache(rows, vocab, element_size(dtype), 128 << 20)};
  OAKE_BY_TYPE(dtype, run_score_grad, p, a, (hipStream_t)stream);
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
  const Plan p = forward_plan(vocab, dtype, 0, top);
  if (blocks_of(p, rows) > kMostBlocks) return refuse(OAKE_ERR_INVALID, "%s: too many rows of this length", what);
  if (int rc = check_scratch(what, d_workspace, workspace_bytes, scratch_bytes(rows, p.sp, 0))) return rc;
  const DistillArgs a{{d_logits, rows, vocab, row_stride, nullptr, 0, scale,
                       past_cache(rows, vocab, element_size(dtype), 256 << 20)}, p.sp,
                      {d_top_indices, d_top_logprobs, index_dtype == OAKE_I64, top, tail != 0}, d_loss, d_stats,
                      static_cast<float*>(d_workspace)};
  OAKE_BY_TYPE(dtype, run_distill, p, a, (hipStream_t)stream);
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
  const Plan p = backward_plan(vocab, dtype, top);
  if (blocks_of(p, rows) > kMostBlocks) return refuse(OAKE_ERR_INVALID, "%s: too many rows of this length", what);
  const DistillGradArgs a{{d_logits, rows, vocab, row_stride, nullptr, 0, scale,
                           past_cache(rows, vocab, element_size(dtype), 256 << 20)}, p.sp,
                          {d_top_indices, d_top_logprobs, index_dtype == OAKE_I64, top, tail != 0},
                          d_stats, d_grad_loss, d_grad, grad_stride,
                          past_cache(rows, vocab, element_size(dtype), 128 << 20)};
  OAKE_BY_TYPE(dtype, run_distill_grad, p, a, (hipStream_t)stream);
  return launched(what);
}

}  // extern "C"

// tokens.hip — operators of token policies: rows of logits over a whole vocabulary instead of the <= 28 actions of pointwise.hip.
//   cbm_top_logits         the K largest logits of each row, their indices, the row's log-sum-exp (what a teacher hands to its student)
//   cbm_distill_loss_grad  distillation from a teacher's top logits: loss and gradient in one call, as cbm_ppo_loss_grad / cbm_impala_loss_grad
//   cbm_verify_drafts      drafted tokens against the target's probabilities (the truncated ratio of cbm_vtrace, per token), and the next token
// All are bound by reading the logits once (the gradient: and writing it once).  Rows start at any element (odd vocabularies): 16-byte loads
// at element alignment, which the load unit takes.  Row statistics are (maximum, sum) pairs: a thread's terms in fp32 (steps of at most 64, up to 2048 in all
// at 2^19 tokens), everything across threads and everything that a decision or a loss depends on in fp64.
#include "cbm_ctx.h"
#include <float.h>
#include <math.h>

namespace {

constexpr int TK_MAX_VOCAB = 1 << 19;   // indices are 19 bits of a key in the top-K kernels; a row's bitmap (one bit a token and a word) is 64 KB of the 160 KB LDS
constexpr int TK_MAX_TOP = 256;         // slots of a row: four a lane of the wave that owns the row's teacher
constexpr int TK_MAX_DRAFTS = 128;      // one thread a draft in the acceptance step
constexpr int TK_MAX_ROWS = 1 << 22;    // a launch holds fewer than 2^32 threads, a row up to 1024

// ------------------------------------------------------------------------------------------ 16 bytes of logits
typedef uint32_t tk_u4 __attribute__((ext_vector_type(4)));
struct Pack { tk_u4 w; };
template <int DT> struct Lg { static constexpr int ES = DT == CBM_F32 ? 4 : 2, VEC = 16 / ES; };
template <int DT> constexpr uint32_t TK_NEG = DT == CBM_F32 ? 0xff800000u : (DT == CBM_BF16 ? 0xff80ff80u : 0xfc00fc00u);   // -inf, twice for 16 bits

__device__ __forceinline__ Pack tk_load16(const char* p) { Pack x; __builtin_memcpy(&x, p, 16); return x; }
__device__ __forceinline__ void tk_store16(char* p, const Pack& x) { __builtin_memcpy(p, &x, 16); }
template <int DT> __device__ __forceinline__ Pack tk_neg() { return Pack{{TK_NEG<DT>, TK_NEG<DT>, TK_NEG<DT>, TK_NEG<DT>}}; }
template <int DT> __device__ __forceinline__ float tk_get(const Pack& p, int j) {
  if constexpr (DT == CBM_F32) return __uint_as_float(p.w[j]);
  const uint32_t w = p.w[j >> 1];
  if constexpr (DT == CBM_BF16) return __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(j & 1 ? w >> 16 : w & 0xffffu));
}
// the largest of a pack's elements, NaN aside
template <int DT> __device__ __forceinline__ float tk_max(const Pack& p) {
  if constexpr (DT == CBM_F16) {             // two at a time
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const uint32_t a = p.w[0], b = p.w[1], c = p.w[2], d = p.w[3];   // (bit_cast of a vector's element would take the first)
    const h2 m = __builtin_elementwise_max(__builtin_elementwise_max(__builtin_bit_cast(h2, a), __builtin_bit_cast(h2, b)),
                                           __builtin_elementwise_max(__builtin_bit_cast(h2, c), __builtin_bit_cast(h2, d)));
    return fmaxf((float)m[0], (float)m[1]);
  } else {
    float m = tk_get<DT>(p, 0);
#pragma unroll
    for (int j = 1; j < Lg<DT>::VEC; ++j) m = fmaxf(m, tk_get<DT>(p, j));
    return m;
  }
}
template <int DT> __device__ __forceinline__ float tk_at(const char* row, int e) {   // one element
  if constexpr (DT == CBM_F32) { float f; __builtin_memcpy(&f, row + (size_t)e * 4, 4); return f; }
  uint16_t h; __builtin_memcpy(&h, row + (size_t)e * 2, 2);
  if constexpr (DT == CBM_BF16) return __uint_as_float((uint32_t)h << 16);
  return (float)__builtin_bit_cast(_Float16, h);
}
// the gradient's one rounding: fp32 -> the logits' type, to nearest even
typedef float tk_f2 __attribute__((ext_vector_type(2)));
typedef __bf16 tk_b2 __attribute__((ext_vector_type(2)));
typedef _Float16 tk_h2 __attribute__((ext_vector_type(2)));
template <int DT> __device__ __forceinline__ void tk_put2(Pack& p, int j, float a, float b) {   // elements j, j+1 (j even)
  if constexpr (DT == CBM_F32) { p.w[j] = __float_as_uint(a); p.w[j + 1] = __float_as_uint(b); }
  else if constexpr (DT == CBM_BF16) p.w[j >> 1] = __builtin_bit_cast(uint32_t, __builtin_convertvector((tk_f2){a, b}, tk_b2));
  else p.w[j >> 1] = __builtin_bit_cast(uint32_t, __builtin_convertvector((tk_f2){a, b}, tk_h2));
}
template <int DT> __device__ __forceinline__ void tk_set(char* row, int e, float v) {
  if constexpr (DT == CBM_F32) __builtin_memcpy(row + (size_t)e * 4, &v, 4);
  else if constexpr (DT == CBM_BF16) { const __bf16 h = (__bf16)v; __builtin_memcpy(row + (size_t)e * 2, &h, 2); }
  else { const _Float16 h = (_Float16)v; __builtin_memcpy(row + (size_t)e * 2, &h, 2); }
}
// keeps the compiler from holding the decoded floats of a resident row from one pass over it to the next (twice the registers, spills at 1024 threads)
__device__ __forceinline__ void tk_redecode(Pack& x) { asm volatile("" : "+v"(x.w)); }
// vector `vi` of a row of V elements, -inf behind its end
template <int DT> __device__ __forceinline__ Pack tk_load(const char* row, int vi, int V) {
  constexpr int VEC = Lg<DT>::VEC, ES = Lg<DT>::ES;
  const int e = vi * VEC;
  if (e + VEC <= V) return tk_load16(row + (size_t)e * ES);
  Pack x = tk_neg<DT>();
  if (e < V) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      if (e + j < V) {
        if constexpr (ES == 4) { uint32_t f; __builtin_memcpy(&f, row + (size_t)(e + j) * 4, 4); x.w[j] = f; }
        else {
          uint16_t h; __builtin_memcpy(&h, row + (size_t)(e + j) * 2, 2);
          x.w[j >> 1] = j & 1 ? (x.w[j >> 1] & 0xffffu) | ((uint32_t)h << 16) : (x.w[j >> 1] & 0xffff0000u) | h;
        }
      }
    }
  }
  return x;
}

__device__ __forceinline__ float tk_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float tk_base(float m) { return m == -INFINITY ? 0.0f : m; }   // what a maximum of -inf is replaced by: exp2(-inf - 0) = 0, not NaN

// 2^((z - b) c), b >= every z: one fma an element, 2^(z c - bc) with bc = fl(b c), what bc was rounded by goes into `fix`, a factor of the whole.  Where b c is so
// large that this would not do (beyond 2^20: the roundings would be powers of two themselves), `far` says so, and exact differences are taken instead,
// in rolled loops that read the row again: masks of a type's lowest values over whole rows come there, and little else.
struct ExpSum {
  float b, c, bc, fix;
  bool far;
  __device__ __forceinline__ ExpSum(float base, float c_) : b(base), c(c_), bc(base * c_), fix(tk_exp2(-fmaf(base, c_, -bc))), far(!(fabsf(bc) <= 0x1p20f)) {}
  __device__ __forceinline__ float operator()(float z) const { return tk_exp2(fmaf(z, c, -bc)); }
  __device__ __forceinline__ float exact(float z) const { return tk_exp2((z - b) * c); }
  template <int DT> __device__ __forceinline__ float sum(const Pack& x) const {
    float p = 0.0f;
#pragma unroll
    for (int j = 0; j < Lg<DT>::VEC; ++j) p += (*this)(tk_get<DT>(x, j));
    return p;
  }
  template <int DT> __device__ __forceinline__ float exact_sum(const Pack& x) const {
    float p = 0.0f;
#pragma unroll
    for (int j = 0; j < Lg<DT>::VEC; ++j) p += exact(tk_get<DT>(x, j));
    return p;
  }
};

// ------------------------------------------------------------------------------------------ reductions
template <class Tp> __device__ __forceinline__ Tp wave_sum(Tp v) { for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64); return v; }
__device__ __forceinline__ float wave_max(float v) { for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64)); return v; }

// (maximum, sum of exp2((z - maximum) c)) of a block's threads: every thread ends with both.  `red` holds a pair a wave.
struct MS { float m; double s; };
template <int T> __device__ __forceinline__ MS block_lse(float m, float s, float c, MS* red) {
  const float wm = wave_max(m), wb = tk_base(wm);
  const double ws = wave_sum((double)(s * tk_exp2((m - wb) * c)));   // (a thread without logits: m = -inf, factor 0)
  if constexpr (T == 64) return MS{wm, ws};
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = MS{wm, ws};
  __syncthreads();
  float M = red[0].m;
#pragma unroll
  for (int i = 1; i < T / 64; ++i) M = fmaxf(M, red[i].m);
  const float B = tk_base(M);
  double S = 0.0;
#pragma unroll
  for (int i = 0; i < T / 64; ++i) S += red[i].s * (double)tk_exp2((red[i].m - B) * c);
  return MS{M, S};
}

// ------------------------------------------------------------------------------------------ distillation from a teacher's top logits
// t_k: the teacher's probabilities of its K slots (softmax over the slots, or exp(v_k / tau - lse) with the tail t_T = 1 - sum t_k), s = softmax(z / tau),
// s_T = sum of s outside the slots' tokens ("top"):
//   loss  = w tau^2 [ sum_k t_k (log t_k - log s_{i_k}) + t_T (log t_T - log s_T) ]
//   dz_j  = w tau   [ s_j (sum_k t_k + t_T) - sum_{k: i_k = j} t_k - [j outside top] t_T s_j / s_T ]
// A block takes a row at a time.  The row's first NV vectors a thread stay in registers, so that the logits are read once for statistics and gradient;
// what lies behind them is read twice.  With a tail, a bitmap of the top tokens keeps them out of the streamed sum: s_T is then a sum of its own with a
// maximum of its own, not a difference that cancels, and the top tokens join it from the wave that holds the teacher.  Every other token's gradient is
// one coefficient times an exponential; the top tokens' gradients are stored last, over what the stream left.
// log2(e) / tau is rounded to fp32 once and used so throughout the student's side, loss included: the loss of a temperature off by 6e-8.
// Bound by memory where there are rows enough: 3840 rows of 131072 bf16, K 64, 427 us = 4.7 TB/s of one reading and one writing (a large copy reaches 4.85),
// the loss alone 217 us = 4.6 TB/s; 777 rows of 50021 fp32 with a tail, a fifth of them padding that is written only, 71 us = 3.9 TB/s (three rows a compute
// unit, and a bit: the last ones are alone).  Small calls are bound by the launch: 3840 rows of 18 actions take 10.6 us, 60 rows of 32768 8.6.  A few rows
// are bound by one block's latency: 1 row of 131072 bf16 18 us, 64 rows 20.  One pass over the row in memory costs a block's own latency (load, statistics,
// barrier, gradient), which the other blocks of a compute unit cover; keeping the next row's loads in flight in the same block needed the registers of a
// second row and was slower (spills).
struct DistillArgs {
  const char* logits; int64_t ld;            // bytes from row to row
  char* grad; int64_t ldg;                   // null: loss only
  const int32_t* idx; const float* val; const float* lse; const float* weight;
  float* loss;
  int rows, V, K;
  float c;                                   // log2(e) / tau
  double inv_tau, tau;
};
// a pack with the elements of `top` (a bit each) at -inf
template <int DT> __device__ __forceinline__ void distill_mask(Pack& x, uint32_t top) {
#pragma unroll
  for (int j = 0; j < Lg<DT>::VEC; ++j) if (top >> j & 1) {
    if constexpr (DT == CBM_F32) x.w[j] = TK_NEG<DT>;
    else x.w[j >> 1] = j & 1 ? (x.w[j >> 1] & 0xffffu) | (TK_NEG<DT> & 0xffff0000u) : (x.w[j >> 1] & 0xffff0000u) | (TK_NEG<DT> & 0xffffu);
  }
}
template <int DT> __device__ __forceinline__ Pack distill_pack(const Pack& x, const ExpSum& es, float coef) {
  Pack g;
#pragma unroll
  for (int j = 0; j < Lg<DT>::VEC; j += 2) tk_put2<DT>(g, j, coef * es(tk_get<DT>(x, j)), coef * es(tk_get<DT>(x, j + 1)));
  return g;
}
template <int DT> __device__ __forceinline__ Pack distill_pack_exact(const Pack& x, const ExpSum& es, float coef) {
  Pack g;
#pragma unroll
  for (int j = 0; j < Lg<DT>::VEC; j += 2) tk_put2<DT>(g, j, coef * es.exact(tk_get<DT>(x, j)), coef * es.exact(tk_get<DT>(x, j + 1)));
  return g;
}
template <int DT, int T, int NV, bool TAIL>
__global__ __launch_bounds__(T) void distill_kernel(DistillArgs a) {
  constexpr int VEC = Lg<DT>::VEC, ES = Lg<DT>::ES, U = 4;
  __shared__ MS red[T / 64];
  __shared__ __align__(16) int32_t sidx[TK_MAX_TOP];
  __shared__ float sz[TK_MAX_TOP], sv[TK_MAX_TOP];     // the student's and the teacher's logits there
  __shared__ double st[TK_MAX_TOP], slt[TK_MAX_TOP];   // t_k and log t_k
  __shared__ uint8_t ssame[TK_MAX_TOP];      // 0: not the first slot of its token (or empty), 1: its only one, 2: the first of several
  __shared__ double steacher[2];             // sum of t_k, t_T
  __shared__ MS stop;                        // TAIL: (maximum, sum) of the student's logits at the top tokens
  extern __shared__ uint32_t bits[];         // TAIL: bit j set: token j is a top token
  const int tid = threadIdx.x, V = a.V, K = a.K;   // (K <= T)
  const int64_t r = blockIdx.x;
  // The row's vectors begin where 16 bytes do (a row of an odd vocabulary starts anywhere); the up to VEC - 1 elements before and behind them are one a thread.
  const char* row0 = a.logits + r * a.ld;
  char* grow0 = a.grad ? a.grad + r * a.ldg : nullptr;
  const int head = min((int)(-(uintptr_t)row0 & 15) / ES, V), nfull = (V - head) / VEC, rem = V - nfull * VEC;
  const char* row = row0 + head * ES;
  char* grow = grow0 + head * ES;
  const int ee = tid < head ? tid : nfull * VEC + tid;   // the thread's single element, where tid < rem
  const float w = a.weight ? a.weight[r] : 1.0f;
  const auto tops = [&](int v) {             // the bits of vector v's elements
    const int e = head + v * VEC;
    return (uint32_t)((((uint64_t)bits[(e >> 5) + 1] << 32) | bits[e >> 5]) >> (e & 31)) & ((1u << VEC) - 1);
  };
  const auto zeros = [&] {                   // a row without a loss
    if (tid == 0) a.loss[r] = 0.0f;
    if (!grow0) return;
    const Pack z = {{0, 0, 0, 0}};
    for (int v = tid; v < nfull; v += T) tk_store16(grow + (size_t)v * 16, z);
    if (tid < rem) tk_set<DT>(grow0, ee, 0.0f);
  };
  if (w == 0.0f) return zeros();             // padding: the row is not looked at

  int my = -1;                               // slot `tid`: its token
  float myv = -INFINITY, myz = -INFINITY;    // the teacher's and the student's logit
  if (tid < K) {
    my = a.idx[r * K + tid];
    myv = a.val[r * K + tid];
  }
  Pack x[NV];                                // the row, as far as it stays; what lies behind its last whole vector is left out where it is used
  if (nfull) {
#pragma unroll
    for (int i = 0; i < NV; ++i) if (i * T < nfull) x[i] = tk_load16(row + (uint32_t)(min(i * T + tid, nfull - 1) * 16));
  }
  const float xe = tid < rem ? tk_at<DT>(row0, ee) : -INFINITY;
  if ((uint32_t)my >= (uint32_t)V) my = -1;  // -1 and whatever lies outside the vocabulary: an empty slot
  if (my >= 0) myz = tk_at<DT>(row0, my);
  if (tid < K) { sidx[tid] = my; sz[tid] = myz; sv[tid] = my >= 0 ? myv : -INFINITY; }
  else if (tid < ((K + 3) & ~3)) sidx[tid] = -2;
  if constexpr (TAIL) for (int i = tid; i < (V + 31) / 32 + 1; i += T) bits[i] = 0;
  __syncthreads();
  if (tid < K) {
    int same = 0, low = K;                   // how many slots hold the token, the first of them
    for (int j = 0; j < K; j += 4) {
      const int4 of = *reinterpret_cast<const int4*>(sidx + j);
      const uint32_t is = (of.x == my ? 1u : 0u) | (of.y == my ? 2u : 0u) | (of.z == my ? 4u : 0u) | (of.w == my ? 8u : 0u);
      same += __popc(is);
      low = min(low, is ? j + (int)__builtin_ctz(is | 16u) : K);
    }
    ssame[tid] = my < 0 || low != tid ? 0 : (same == 1 ? 1 : 2);
    if constexpr (TAIL) if (my >= 0) atomicOr(&bits[my >> 5], 1u << (my & 31));
  }
  if constexpr (TAIL) __syncthreads();
  if (tid < 64) {                        // t_k in fp64, and the top tokens' own (maximum, sum), each token once: beside the other waves' statistics
    float vm = -INFINITY;
    for (int k = tid; k < K; k += 64) vm = fmaxf(vm, sv[k]);
    const double at = TAIL ? (double)a.lse[r] : (double)tk_base(wave_max(vm)) * a.inv_tau;
    double sum = 0.0;
    for (int k = tid; k < K; k += 64) {
      const double lt = (double)sv[k] * a.inv_tau - at, t = sv[k] == -INFINITY ? 0.0 : exp(lt);
      st[k] = t; slt[k] = lt;
      sum += t;
    }
    sum = wave_sum(sum);
    if (!TAIL && sum > 0.0) {
      const double ls = log(sum), inv = 1.0 / sum;
      for (int k = tid; k < K; k += 64) { st[k] *= inv; slt[k] -= ls; }
      sum = 1.0;
    }
    bool filled = false;                     // (a teacher without a slot has no tail either)
    if constexpr (TAIL) for (int k = tid; k < K; k += 64) filled |= ssame[k] != 0;
    filled = __any(filled);
    if (tid == 0) { steacher[0] = sum; steacher[1] = TAIL && filled ? (sum > 1.0 ? 0.0 : 1.0 - sum) : 0.0; }
    if constexpr (TAIL) {
      float zm = -INFINITY;
      for (int k = tid; k < K; k += 64) if (ssame[k]) zm = fmaxf(zm, sz[k]);
      zm = wave_max(zm);
      double zs = 0.0;
      for (int k = tid; k < K; k += 64) if (ssame[k]) zs += exp2(((double)sz[k] - (double)tk_base(zm)) * (double)a.c);
      zs = wave_sum(zs);
      if (tid == 0) stop = MS{zm, zs};
    }
  }
  // statistics of the row (TAIL: of what lies outside top)
  float m = xe;
  if constexpr (TAIL) if (tid < rem) { if (bits[ee >> 5] >> (ee & 31) & 1) m = -INFINITY; }
  const float xs = m;
  int t = cbm_opaque_vgpr(tid);          // (or the compiler keeps NV places and masks from pass to pass, in registers that the row needs)
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (i * T >= nfull) continue;            // (the same for every thread)
    const int v = i * T + t;
    if constexpr (TAIL) { const uint32_t top = tops(max(min(v, nfull - 1), 0)); if (top) distill_mask<DT>(x[i], top); }
    const float vm = tk_max<DT>(x[i]);
    m = v < nfull ? fmaxf(m, vm) : m;
    tk_redecode(x[i]);
  }
  const ExpSum es(tk_base(m), a.c);
  float s = tk_exp2((xs - es.b) * a.c), p = 0.0f;
  t = cbm_opaque_vgpr(tid);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (i * T >= nfull) continue;
    const float q = es.sum<DT>(x[i]);
    p += i * T + t < nfull ? q : 0.0f;
    tk_redecode(x[i]);
  }
  s += es.far ? 0.0f : p * es.fix;
  for (int v0 = (es.far ? 0 : NV * T) + tid; v0 < nfull; v0 += U * T) {   // what does not stay: running maximum and sum, U vectors in flight
    Pack y[U];
    float nm = m;
#pragma unroll
    for (int u = 0; u < U; ++u) y[u] = tk_load16(row + (uint32_t)(min(v0 + u * T, nfull - 1) * 16));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = v0 + u * T;
      if constexpr (TAIL) { const uint32_t top = tops(min(v, nfull - 1)); if (top) distill_mask<DT>(y[u], top); }
      const float vm = tk_max<DT>(y[u]);
      nm = v < nfull ? fmaxf(nm, vm) : nm;
      tk_redecode(y[u]);
    }
    const ExpSum ey(tk_base(nm), a.c);
    float q = 0.0f;
    if (!ey.far) {
#pragma unroll
      for (int u = 0; u < U; ++u) { const float e = ey.sum<DT>(y[u]); q += v0 + u * T < nfull ? e : 0.0f; }
      q *= ey.fix;
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) { const float e = ey.exact_sum<DT>(y[u]); q += v0 + u * T < nfull ? e : 0.0f; }
    }
    s = s * tk_exp2((m - ey.b) * a.c) + q;
    m = nm;
  }
  const MS ms = block_lse<T>(m, s, a.c, red);
  if constexpr (T == 64) __syncthreads();   // (a wider block has passed one in block_lse)
  // the whole row's statistics, and the coefficient of the tokens outside top
  float M = ms.m;
  double S = ms.s, tT = 0.0;
  const double sumT = steacher[0];
  if constexpr (TAIL) {
    M = fmaxf(ms.m, stop.m);
    const float B = tk_base(M);
    S = ms.s * (double)tk_exp2((ms.m - B) * a.c) + stop.s * (double)tk_exp2((stop.m - B) * a.c);
    tT = ms.m == -INFINITY ? 0.0 : steacher[1];   // no logit outside top: the tail is left out
  }
  if (S == 0.0 || (sumT == 0.0 && steacher[1] == 0.0)) return zeros();   // nothing in the student's row, or nothing in the teacher's (the same for every thread)
  if (tid < 64) {
    // With a tail, an error of s_T that is in the whole's sum too meets s_T - t_T only; one of the factor that takes it there meets 1: that factor in fp64.
    const double whole = TAIL ? ms.s * exp2(((double)ms.m - (double)tk_base(M)) * (double)a.c) + stop.s * exp2(((double)stop.m - (double)tk_base(M)) * (double)a.c) : S;
    const double logS = log(whole), lc = (double)a.c * 0.69314718055994530942;
    double l = 0.0;
    for (int k = tid; k < K; k += 64) if (st[k] != 0.0) l += st[k] * (slt[k] - (((double)sz[k] - (double)M) * lc - logS));
    l = wave_sum(l);
    if (tid == 0) {
      if (tT > 0.0) l += tT * (log(tT) - (((double)ms.m - (double)M) * lc + log(ms.s) - logS));
      a.loss[r] = (float)((double)w * a.tau * a.tau * l);
    }
  }
  if (!grow0) return;
  const double wt = (double)w * a.tau;
  float ref, coef;
  if constexpr (TAIL) {
    ref = tk_base(ms.m);                     // 2^((z - ref) c) <= 1 for every token outside top
    const double sT = ms.s * (double)tk_exp2((ms.m - tk_base(M)) * a.c) / S;   // their probability
    coef = ms.m == -INFINITY ? 0.0f : (float)(wt * ((sumT + tT) * sT - tT) / ms.s);
  } else {
    ref = tk_base(M);
    coef = (float)(wt * sumT / S);
  }
  // (an infinite 2^.. of a top token is overwritten below; a NaN in the row has made coef NaN)
  const ExpSum eg(ref, a.c);
  if (!eg.far) {
    const float cf = coef * eg.fix;
    t = cbm_opaque_vgpr(tid);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i * T >= nfull) continue;
      tk_redecode(x[i]);
      const Pack g = distill_pack<DT>(x[i], eg, cf);
      if (i * T + t < nfull) tk_store16(grow + (uint32_t)((i * T + t) * 16), g);
    }
  }
  for (int v0 = (eg.far ? 0 : NV * T) + tid; v0 < nfull; v0 += U * T) {
    Pack y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) y[u] = tk_load16(row + (uint32_t)(min(v0 + u * T, nfull - 1) * 16));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Pack g = eg.far ? distill_pack_exact<DT>(y[u], eg, coef) : distill_pack<DT>(y[u], eg, coef * eg.fix);
      if (v0 + u * T < nfull) tk_store16(grow + (uint32_t)((v0 + u * T) * 16), g);
    }
  }
  if (tid < rem) tk_set<DT>(grow0, ee, coef * eg.exact(xe));
  __syncthreads();                           // the stream's stores come before the top tokens'
  if (tid < K && ssame[tid]) {
    double d = st[tid];
    if (ssame[tid] == 2) for (int j = tid + 1; j < K; ++j) if (sidx[j] == my) d += st[j];   // a token in several slots: all of their t_k
    const double sk = (double)tk_exp2((myz - tk_base(M)) * a.c) / S;
    tk_set<DT>(grow0, my, (float)(wt * (sk * (sumT + tT) - d)));
  }
}

template <int DT, int T, int NV>
void distill_launch(const DistillArgs& a, hipStream_t st) {
  if (a.lse) hipLaunchKernelGGL((distill_kernel<DT, T, NV, true>), dim3(a.rows), dim3(T), ((a.V + 31) / 32 + 1) * 4, st, a);
  else hipLaunchKernelGGL((distill_kernel<DT, T, NV, false>), dim3(a.rows), dim3(T), 0, st, a);
}
// 8 vectors a thread stay (80 registers); 6 blocks of 256 threads share a compute unit, 3 of 512, and one of 1024 is alone there: the loads, sums and stores of
// neighbours overlap.  A larger block reads less of its row twice, a smaller one has more company.  3840 rows with gradient, us by blocks of 256 / 512 / 1024:
// 20000 bf16 (2500 vectors) 70 / 86 / 144, 32768 bf16 122 / 106 / 170, 65536 bf16 (8192) 260 / 216 / 251, 50021 fp32 (12506) 453 / 358 / 325,
// 131072 bf16 (16384) 575 / 470 / 427.  (Fewer rows go by the same rule.)  12 or 16 vectors a thread: 424 and 442 there, 320 and 318 at 50021 fp32.  K <= T.
template <int DT>
void distill_dispatch(const DistillArgs& a, hipStream_t st) {
  const int nv = (a.V + Lg<DT>::VEC - 1) / Lg<DT>::VEC;
  if (nv <= 64 && a.K <= 64) distill_launch<DT, 64, 1>(a, st);
  // (16384 rows, bf16, K 64, us: 1000 tokens 33 by a wave, 74 by 256 threads; 4000 tokens, K 64, 59 by two waves, 88 by 256 threads)
  else if (nv <= 256 && a.K <= 64) distill_launch<DT, 64, 4>(a, st);
  else if (nv <= 512 && a.K <= 128) distill_launch<DT, 128, 4>(a, st);
  else if (nv <= 10 * 256) distill_launch<DT, 256, 8>(a, st);
  else if (nv <= 20 * 512) distill_launch<DT, 512, 8>(a, st);
  else distill_launch<DT, 1024, 8>(a, st);
}

// ------------------------------------------------------------------------------------------ the K largest logits of a row
// Keys: (order of the fp32 value, 19 bits of 2^19 - 1 - index): unique, and their order is "larger value first, equal values by rising index".
// A block streams its row (or its share of one: few rows are split and joined) in chunks of EPT elements a thread, with the running maximum and
// sum a thread for the log-sum-exp, and appends what is above a bar to a buffer in LDS.  The first bar comes from the first chunk: the K-th largest
// of the threads' maxima has K elements at or above it, and with T >= 2 K threads few more (1.2 to 1.4 K of random data).  After the 2nd, 4th, 8th .. chunk the
// K-th largest key of the buffer raises it, so that a row of n chunks appends about K (1 + log2 n) keys.  An element that only equals the bar comes
// behind K others and is left out.  Should the buffer overflow all the same (rising rows), the lanes that found no room wait while it is cut to T keys,
// and a chunk that alone would fill it is held to the exact K-th of its threads' maxima: K threads, EPT K keys, the room there is.
// 3840 rows of 32768 bf16, K 32: 66 us = 3.8 TB/s, 1009 of 100003 fp16 at odd addresses, K 128: 65 us = 3.1 TB/s.  Counted there: 13.7 and 13.4 vector
// instructions an element (it is decoded for the maximum and for the sum), the vector units busy for 67 and 51 % of the time: 16-bit rows are bound by them and
// by the barriers of a block (first bar, cuts, order), which with K 128 have 14.6 waves a compute unit to hide behind.  Short rows with large K are bound by
// the buffer: choosing the bar and ordering K keys (each counts those above it, n^2 / 64 comparisons a block).  16384 rows of 1000: K 8 20 us, K 64 46,
// K 256 364 (vector units busy for 60 % of it, LDS for 56).
struct TopArgs {
  const char* logits; int64_t ld;
  int32_t* idx; float* val; float* lse;
  uint64_t* ws_keys; MS* ws_ms;              // with nsplit > 1: [row][split][K] and [row][split]
  int V, K, nsplit, cap, rows;               // cap = EPT K + T keys
  float c;
  double inv_tau;
};
__device__ __forceinline__ uint32_t top_order(float v) {   // unsigned order of the values; -0 becomes +0
  const uint32_t u = __float_as_uint(v + 0.0f);
  return u ^ (uint32_t)(((int32_t)u >> 31) | (int32_t)0x80000000);
}
__device__ __forceinline__ float top_value(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }
__device__ __forceinline__ float top_below(uint32_t o) { return o == 0x80000000u ? __uint_as_float(0x80000001u) : top_value(o - 1); }   // the next smaller number (of 0: of -0 too)
__device__ __forceinline__ uint64_t top_key(float v, int e) { return ((uint64_t)top_order(v) << 19) | (uint32_t)(TK_MAX_VOCAB - 1 - e); }
__device__ __forceinline__ int top_index(uint64_t key) { return TK_MAX_VOCAB - 1 - (int)(key & (TK_MAX_VOCAB - 1)); }
__device__ __forceinline__ uint32_t top_order_of(uint64_t key) { return (uint32_t)(key >> 19); }
constexpr int TOP_KEY_BITS = 51;
constexpr int TOP_SPLIT_T = 256;             // the threads of a block where rows are split (top_plan)

// the largest bound that K of the block's T numbers (0: none) reach, or 0 where fewer are there; the first wave's work.  With slack, any bound that K .. K + slack
// of them reach: a third of the steps.
template <int T, class Num> __device__ Num top_bound(Num mine, int bits, int K, int slack, Num* all, Num* sbound) {
  all[threadIdx.x] = mine;
  __syncthreads();
  if (threadIdx.x < 64) {
    Num k[T / 64];
#pragma unroll
    for (int i = 0; i < T / 64; ++i) k[i] = all[i * 64 + threadIdx.x];
    Num b = 0;
    for (int bit = bits - 1; bit >= 0; --bit) {
      const Num cand = b | ((Num)1 << bit);
      int n = 0;
#pragma unroll
      for (int i = 0; i < T / 64; ++i) n += __popcll(__ballot(k[i] >= cand));
      if (n >= K) { b = cand; if (n <= K + slack) break; }
    }
    if (threadIdx.x == 0) *sbound = b;
  }
  __syncthreads();
  const Num b = *sbound;
  __syncthreads();
  return b;
}
template <int T> struct TopShared { uint64_t all[T]; uint64_t bound; int fill; };
// the buffer's n <= MOST T keys (0: none) cut to the K largest and at most `most` (K <= most <= T) in all; returns their number and raises the bar
template <int T, int MOST> __device__ int top_cut(uint64_t* buf, int n, int K, int most, float* bar, TopShared<T>& sh) {
  // Of n > T keys, ceil(n / T) a thread, an exact cut leaves ceil(n / T) K, as T >= 2 K at most half and a bit: 8 turns are more than it takes.
  for (int turn = 0; n > most && turn < 8; ++turn) {
    uint64_t k[MOST], best = 0;
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
      k[i] = i * T + (int)threadIdx.x < n ? buf[i * T + threadIdx.x] : 0;
      best = k[i] > best ? k[i] : best;
    }
    uint64_t bound;                          // (its barriers stand between the reads above and the writes below)
    if (turn > 0) bound = top_bound<T, uint64_t>(best, TOP_KEY_BITS, K, 0, sh.all, &sh.bound);   // (equal values may have kept too many: now their indices tell them apart)
    else bound = (uint64_t)top_bound<T, uint32_t>(top_order_of(best), 32, K, K / 4, (uint32_t*)sh.all, (uint32_t*)&sh.bound) << 19;
    if (bound) *bar = fmaxf(*bar, top_value(top_order_of(bound)));
    if (threadIdx.x == 0) sh.fill = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MOST; ++i) if (k[i] != 0 && k[i] >= bound) buf[atomicAdd(&sh.fill, 1)] = k[i];
    __syncthreads();
    n = sh.fill;
    __syncthreads();
  }
  return n;
}
// writes the buffer's K largest in order; n <= T
template <int T> __device__ void top_write(const uint64_t* buf, int n, int K, int32_t* idx, float* val, uint64_t* keys) {
  const uint64_t mine = (int)threadIdx.x < n ? buf[threadIdx.x] : 0;   // (n <= T; a 0 is no key)
  const int live = __syncthreads_count(mine != 0);
  if (mine) {
    int rank = 0;
    int j = 0;
#pragma unroll 2
    for (; j + 4 <= n; j += 4) {
      const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(buf + j), y = *reinterpret_cast<const ulonglong2*>(buf + j + 2);
      rank += (x.x > mine) + (x.y > mine) + (y.x > mine) + (y.y > mine);
    }
    for (; j < n; ++j) rank += buf[j] > mine;
    if (rank < K) {
      if (keys) keys[rank] = mine;
      else { idx[rank] = top_index(mine); val[rank] = top_value(top_order_of(mine)); }
    }
  }
  for (int k = live + (int)threadIdx.x; k < K; k += T) {
    if (keys) keys[k] = 0;
    else { idx[k] = -1; val[k] = -INFINITY; }
  }
}
__device__ __forceinline__ float top_lse(MS ms, double inv_tau) {
  if (ms.m == -INFINITY && ms.s == 0.0) return -INFINITY;
  if (ms.m == INFINITY) return INFINITY;
  return (float)((double)tk_base(ms.m) * inv_tau + log(ms.s));
}

// a chunk's vectors of a thread; -inf behind the row's last whole vector
template <int DT, int T, int U> __device__ __forceinline__ void top_chunk(Pack (&y)[U], const char* row, int ch, int nfull) {
#pragma unroll
  for (int u = 0; u < U; ++u) y[u] = tk_load16(row + (size_t)min((ch * U + u) * T + (int)threadIdx.x, nfull - 1) * 16);
  if ((ch + 1) * T * U > nfull) {
#pragma unroll
    for (int u = 0; u < U; ++u) if ((ch * U + u) * T + (int)threadIdx.x >= nfull) y[u] = tk_neg<DT>();
  }
}
template <int DT, int T, int EPT, int G, int MOST>
__global__ __launch_bounds__(T) void top_kernel(TopArgs a) {
  constexpr int VEC = Lg<DT>::VEC, U = EPT / VEC;
  extern __shared__ __align__(16) uint64_t buf[];          // [cap]
  __shared__ TopShared<T> sh;
  __shared__ MS red[T / 64];
  __shared__ int sfull[3];                   // whether a chunk's elements found no room: one a pass, in turn
  const int tid = threadIdx.x, V = a.V, K = a.K;
  const int64_t r = blockIdx.x / (uint32_t)a.nsplit;
  const int split = (int)(blockIdx.x - r * a.nsplit);
  // the row's vectors begin where 16 bytes do; the up to VEC - 1 elements before and behind them are one a thread of the last split
  const char* row0 = a.logits + r * a.ld;
  const int head = (int)(-(uintptr_t)row0 & 15) / Lg<DT>::ES, nfull = (V - head) / VEC, rem = V - nfull * VEC, nchunk = (nfull + T * U - 1) / (T * U);   // (V > 64: there are whole vectors)
  const char* row = row0 + head * Lg<DT>::ES;
  const int c0 = (int)((int64_t)nchunk * split / a.nsplit), c1 = (int)((int64_t)nchunk * (split + 1) / a.nsplit);
  const int ee = tid < head ? tid : nfull * VEC + tid;
  const float extra = split == a.nsplit - 1 && tid < rem ? tk_at<DT>(row0, ee) : -INFINITY;
  Pack x[G][U];                              // G chunks at a time: one bar, one maximum, one rescaling for all; each chunk's registers take the next group's as it is done
#pragma unroll
  for (int g = 0; g < G; ++g) top_chunk<DT, T, U>(x[g], row, c0 + g < c1 ? c0 + g : nchunk, nfull);
  if (tid == 0) sh.fill = 0;
  if (tid < 3) sfull[tid] = 0;
  float bar = -INFINITY;                     // an element has to be above it
  float m = extra, s = extra == -INFINITY ? 0.0f : tk_exp2(extra - extra);   // 1, or NaN
  int turn = 0, done = 0;
  __syncthreads();
  for (int c = c0; c < c1; c += G) {
    float vm[G][U], cm = -INFINITY;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        vm[g][u] = -INFINITY;
        if (((c + g) * U + u) * T >= nfull) continue;   // (the same for every thread: short rows do not fill a group)
        vm[g][u] = tk_max<DT>(x[g][u]);
        cm = fmaxf(cm, vm[g][u]);
        tk_redecode(x[g][u]);
      }
    const float nm = fmaxf(m, cm);
    const ExpSum es(tk_base(nm), a.c);
    float p = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (((c + g) * U + u) * T >= nfull) continue;
        p += es.sum<DT>(x[g][u]);
        tk_redecode(x[g][u]);
      }
    p *= es.fix;
    if (es.far) {
      p = 0.0f;
#pragma unroll 1
      for (int q = 0; q < G * U; ++q) { const int v = (c * U + q) * T + tid; if (c + q / U < c1 && v < nfull) p += es.exact_sum<DT>(tk_load16(row + (size_t)v * 16)); }
    }
    s = s * tk_exp2((m - es.b) * a.c) + p;
    m = nm;
    float over = bar;                        // what an element of this group has to be above: just below the bar while equal ones may come before those that made it
    if (c == c0) {
      const uint32_t o = top_bound<T, uint32_t>(cm > -INFINITY ? top_order(cm) : 0u, 32, K, K / 4, (uint32_t*)sh.all, (uint32_t*)&sh.bound);
      if (o) { bar = top_value(o); over = top_below(o); }
    }
    uint32_t wait[G];                        // the thread's elements that are above, a bit each
#pragma unroll
    for (int g = 0; g < G; ++g) {
      wait[g] = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!(vm[g][u] > over)) continue;
        uint32_t bits = 0;
#pragma unroll
        for (int q = VEC - 1; q >= 0; --q) bits = bits + bits + (tk_get<DT>(x[g][u], q) > over ? 1u : 0u);
        wait[g] |= bits << (u * VEC);
      }
      if (c + G < c1) top_chunk<DT, T, U>(x[g], row, c + G + g < c1 ? c + G + g : nchunk, nfull);
    }
    // appends those that reach the bound; what finds no room stays.  (Elements again from memory: an indexed register would cost more, and hits are few.)
    const auto append = [&](uint32_t waits, int ch, uint64_t bound) {
      uint32_t left = 0;
      for (uint32_t w = waits; w; w &= w - 1) {
        const int q = __builtin_ctz(w), e = ((ch * U + q / VEC) * T + tid) * VEC + q % VEC;
        const float z = tk_at<DT>(row, e);
        const uint64_t k = top_key(z, head + e);
        if (z > over && k >= bound) {
          const int at = atomicAdd(&sh.fill, 1);
          if (at < a.cap) buf[at] = k;
          else left |= 1u << q;
        }
      }
      return left;
    };
    bool any = false;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (wait[g]) wait[g] = append(wait[g], c + g, 0);
      any |= wait[g] != 0;
    }
    if (any) sfull[turn] = 1;
    __syncthreads();
    const bool full = sfull[turn] != 0;      // (the same for every thread: this turn's flag is written before the barrier only)
    if (tid == 0) sfull[turn == 0 ? 2 : turn - 1] = 0;   // the turn before: read by all before this barrier, written again behind the next but one
    turn = turn == 2 ? 0 : turn + 1;
    if (full) {                              // chunk by chunk: cut, then what reaches the exact K-th of the waiting maxima fits
#pragma unroll 1
      for (int g = 0; g < G; ++g) {
        uint32_t w = wait[0];
#pragma unroll
        for (int q = 1; q < G; ++q) w = q == g ? wait[q] : w;
        const int fill = min(sh.fill, a.cap);
        __syncthreads();
        top_cut<T, MOST>(buf, fill, K, T, &bar, sh);
        over = top_below(top_order(bar));
        uint64_t best = 0;
        for (uint32_t v = w; v; v &= v - 1) {
          const int q = __builtin_ctz(v), e = (((c + g) * U + q / VEC) * T + tid) * VEC + q % VEC;
          const float z = tk_at<DT>(row, e);
          const uint64_t k = top_key(z, head + e);
          if (z > over && k > best) best = k;
        }
        const uint64_t bound = top_bound<T, uint64_t>(best, TOP_KEY_BITS, K, 0, sh.all, &sh.bound);   // (0: fewer than K threads wait, all they hold fits)
        append(w, c + g, bound);
        __syncthreads();
      }
    }
    ++done;
    if (done > 1 && (done & (done - 1)) == 0 && c + G < c1) {   // what the buffer says about the bar
      const int fill = sh.fill;              // (no appends before top_bound's barriers)
      uint32_t o = tid < fill ? top_order_of(buf[tid]) : 0u;
      if (tid + T < fill) { const uint32_t o2 = top_order_of(buf[tid + T]); o = o2 > o ? o2 : o; }
      o = top_bound<T, uint32_t>(o, 32, K, K / 4, (uint32_t*)sh.all, (uint32_t*)&sh.bound);
      if (o) bar = fmaxf(bar, top_value(o));
    }
  }
  __syncthreads();
  int fill = sh.fill;
  __syncthreads();
  fill = top_cut<T, MOST>(buf, fill, K, 3 * K + 32 < T ? 3 * K + 32 : T, &bar, sh);
  if (rem && split == a.nsplit - 1) {        // (cap has room for EPT K more than T)
    if (extra > -INFINITY && extra >= bar) buf[atomicAdd(&sh.fill, 1)] = top_key(extra, ee);   // (those before the vectors count where they equal the bar)
    __syncthreads();
    fill = sh.fill;
    __syncthreads();
    fill = top_cut<T, MOST>(buf, fill, K, T, &bar, sh);
  }
  const MS ms = block_lse<T>(m, s, a.c, red);
  if (T == TOP_SPLIT_T && a.nsplit > 1) {
    top_write<T>(buf, fill, K, nullptr, nullptr, a.ws_keys + (r * a.nsplit + split) * K);
    if (tid == 0) a.ws_ms[r * a.nsplit + split] = ms;
  } else {
    top_write<T>(buf, fill, K, a.idx + r * K, a.val + r * K, nullptr);
    if (tid == 0) a.lse[r] = top_lse(ms, a.inv_tau);
  }
}
// the splits of a row: their keys are one more buffer to cut
template <int T, int MOST>
__global__ __launch_bounds__(T) void top_join_kernel(TopArgs a) {
  extern __shared__ __align__(16) uint64_t buf[];
  __shared__ TopShared<T> sh;
  const int tid = threadIdx.x, K = a.K, n = a.nsplit * K;
  const int64_t r = blockIdx.x;
  for (int i = tid; i < n; i += T) buf[i] = a.ws_keys[r * n + i];
  if (tid < 64) {
    MS ms = tid < a.nsplit ? a.ws_ms[r * a.nsplit + tid] : MS{-INFINITY, 0.0};
    const float M = wave_max(ms.m);
    const double S = wave_sum(ms.s * (double)tk_exp2((ms.m - tk_base(M)) * a.c));
    if (tid == 0) a.lse[r] = top_lse(MS{M, S}, a.inv_tau);
  }
  __syncthreads();
  float bar = -INFINITY;
  int fill = top_cut<T, MOST>(buf, n, K, 3 * K + 32 < T ? 3 * K + 32 : T, &bar, sh);
  top_write<T>(buf, fill, K, a.idx + r * K, a.val + r * K, nullptr);
}

// A vocabulary of a few tokens (an action set): one token a lane, G lanes a row, 64 / G rows a wave; a token's place is the number of tokens before it.
// 15360 rows of 18: 8 us, of which 1.6 MB are 0.4: the launch, then 18 shuffles.
template <int DT, int G>
__global__ __launch_bounds__(256) void top_small_kernel(TopArgs a) {
  const int64_t r = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  const int e = threadIdx.x % G, V = a.V, K = a.K;
  if (r >= a.rows) return;
  const float z = e < V ? tk_at<DT>(a.logits + r * a.ld, e) : -INFINITY;
  float m = z;
  for (int o = G / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, G));
  float s = tk_exp2((z - tk_base(m)) * a.c);
  for (int o = G / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, G);
  const uint32_t mine = z > -INFINITY ? top_order(z) : 0u;   // (a NaN is not above -inf)
  int rank = 0, n = 0;
  for (int j = 0; j < V; ++j) {
    const uint32_t o = (uint32_t)__shfl((int)mine, j, G);
    rank += o > mine || (o == mine && j < e);
    n += o != 0;
  }
  if (mine && rank < K) { a.idx[r * K + rank] = e; a.val[r * K + rank] = z + 0.0f; }
  for (int k = n + e; k < K; k += G) { a.idx[r * K + k] = -1; a.val[r * K + k] = -INFINITY; }
  if (e == 0) a.lse[r] = top_lse(MS{m, (double)s}, a.inv_tau);
}

struct TopPlan { int threads, nsplit, cap; size_t lds, ws; };
int top_ept(int threads, int V) { return threads == 256 ? 32 : (threads == 512 && V <= 4096 ? 8 : 16); }
TopPlan top_plan(int rows, int V, int K) {
  TopPlan p = {};
  p.nsplit = 1;
  if (V <= 64) return p;                     // top_small_kernel
  // T >= 2 K: a chunk's bar leaves 1.4 K of random data above it at most.  T >= 4 K (1.2 K) has fewer blocks on a compute unit: 3840 rows of 100003 fp16,
  // K = 128, by 512 threads 299 us, by 256 221; 131072 bf16, K = 256, by 1024 558, by 512 372; fp32 and smaller K the same
  p.threads = K <= 32 && V <= 1024 ? 64 : (K <= 64 && V <= 2048 ? 128 : (K <= 128 ? 256 : 512));
  // Few rows leave compute units empty: up to 128 long ones are split until there are about 512 blocks, and joined (a second kernel); up to 255 others go to
  // wider blocks.  The border of 49152 tokens lies between the measured 32768 and 100003.  us split / not: 60 x 32768 bf16, K = 32, 20 / 15;
  // 1 x 131072 bf16, K = 64, 21 / 30; 60 of them 21 / 31, 200 34 / 34; 1 x 100003 fp16, K = 128, 27 / 31, 200 39 / 36; K = 256
  // (by 512 threads either way) 1 x 131072 38 / 40, 60 58 / 40.
  const bool split = rows <= 128 && V > 49152 && p.threads == TOP_SPLIT_T;   // (K <= 128)
  if (!split && rows < 256 && V > 16384) p.threads = 512;
  p.cap = top_ept(p.threads, V) * K + p.threads;
  if (split) {
    const int chunk = p.threads * top_ept(p.threads, V), nchunk = (V + chunk - 1) / chunk, n = (512 + rows - 1) / rows;
    p.nsplit = n < nchunk ? n : nchunk;
    p.nsplit = p.nsplit < 16 ? p.nsplit : 16;   // (the join holds nsplit K <= cap keys)
  }
  p.lds = (size_t)p.cap * 8;
  p.ws = p.nsplit > 1 ? (size_t)rows * p.nsplit * ((size_t)K * 8 + sizeof(MS)) : 0;
  return p;
}
template <int DT, int T, int EPT, int G, int KMAX> void top_launch(const TopArgs& a, const TopPlan& p, hipStream_t st) {
  static_assert(2 * KMAX <= T, "or top_cut does not end");
  constexpr int MOST = EPT * KMAX / T + 1;   // cap <= MOST T
  hipLaunchKernelGGL((top_kernel<DT, T, EPT, G, MOST>), dim3((uint32_t)a.rows * p.nsplit), dim3(T), p.lds, st, a);
  if constexpr (T == TOP_SPLIT_T) if (p.nsplit > 1) hipLaunchKernelGGL((top_join_kernel<T, MOST>), dim3(a.rows), dim3(T), p.lds, st, a);
}
template <int DT, int G> void top_launch_small(const TopArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((top_small_kernel<DT, G>), dim3((uint32_t)(((int64_t)a.rows * G + 255) / 256)), dim3(256), 0, st, a);
}
template <int DT> void top_dispatch(const TopArgs& a, const TopPlan& p, hipStream_t st) {
  if (a.V <= 16) top_launch_small<DT, 16>(a, st);
  else if (a.V <= 32) top_launch_small<DT, 32>(a, st);
  else if (a.V <= 64) top_launch_small<DT, 64>(a, st);
  else if (p.threads == 64) top_launch<DT, 64, 16, 1, 32>(a, p, st);
  else if (p.threads == 128) top_launch<DT, 128, 16, 1, 64>(a, p, st);
  else if (p.threads == 256 && a.K <= 64) top_launch<DT, 256, 32, Lg<DT>::VEC / 4, 64>(a, p, st);
  else if (p.threads == 256) top_launch<DT, 256, 32, Lg<DT>::VEC / 4, 128>(a, p, st);
  else if (a.V <= 4096) top_launch<DT, 512, 8, 1, 256>(a, p, st);
  else top_launch<DT, 512, 16, 4, 256>(a, p, st);
}

// ------------------------------------------------------------------------------------------ drafted tokens against the target
// p_i = softmax(target row i / tau), q_i = softmax(draft row i / tau), or one-hot at the drafted token where there are no draft logits.
//   accepted while u_i q_i(x_i) < p_i(x_i), i < n;  at the first rejection a the next token is drawn from max(p_a - q_a, 0) (from p_a where that has
//   no mass), after n acceptances from p_n: the first token whose cumulative weight exceeds u_s times the whole.
// The drawn token lies between two neighbours of a cumulative sum over the whole vocabulary: sums that are off by 1e-7 would move one token in a few
// hundred, so that the row it is drawn from is summed in fp64, exponentials too.  They are 2^(z C - E), C = log2(e) / tau, with a whole number E a chunk of
// 2048 tokens (the maximum's exponent, rounded up): sums of different chunks are brought together by exact shifts of the exponent.  An acceptance compares
// two numbers, and sums of fp32 exponentials do for it where the two are not next to each other (vf_accept).
// Rows of one chunk and few drafts, one kernel:
//   verify_one_kernel             a block a sequence: its rows' sums, then all that follows
// Small calls, two kernels (launches are what they cost):
//   verify_sums_kernel<VF_SUMS>   fp64 sums of each chunk of each row that a sequence may need (a wave a chunk), and of the chunks of a block together
//   verify_pick_kernel<VF_SUMS>   acceptance, by every block of a sequence for itself; where it ends in a rejection with a draft distribution the chunks' sums of
//                                 max(p - q, 0), and the sequence's last block to finish draws the token; elsewhere its first block draws from the sums there are
// Large calls, three kernels (an fp64 exponential is 20 instructions, an fp32 one with its sum 6, and but two rows a sequence need the former):
//   verify_stats_kernel           (maximum, sum) in fp32 of the drafted positions' rows
//   verify_sums_kernel<VF_STATS>  acceptance, and the fp64 sums of the one or two rows that the token is drawn from
//   verify_pick_kernel<VF_STATS>  the rest as above
// Bound: at 64 sequences of up to 8 drafts, 131072 bf16, 79 us a call.  Statistics 29 (134 MB where lengths are 4 in the mean, 268 at most; rows behind n_draft are
// unread): 4.6 TB/s.  Sums 23 and pick 29 (17 MB of target rows, and as much of draft rows where all end in a rejection): an fp64 exponential is 20 instructions, fp64 at the rate of
// unpacked fp32, which keeps the vector units busy for 44 and 20 % of the time; the rest is the chain acceptance, chunk sums, last block, scan, token, with a
// chunk or two a wave behind it.  One sequence of 4 drafts: sums 6, pick 14 to 18 (that chain alone).  37 sequences of 5 looked-up drafts, 50021 fp16:
// 13 and 15.  120 sequences of 7, 18 actions: one kernel, 9.  No drafts, 131072 bf16: one sequence 6 + 15, 64 11 + 14.  Greedy, 64 sequences of up to 8: 23 + 6.
constexpr int VF_T = 256, VF_WAVES = VF_T / 64, VF_CHUNK = 2048;   // 32 tokens a lane: what a chunk costs beside its exps (reductions) is shared by that many
enum { VF_STATS, VF_SUMS, VF_ONE };          // three kernels, two, one
struct VfSum { double e, s; };               // s 2^e; nothing: s = 0, e = -inf; a NaN among the logits: s NaN; +inf: e = +inf
struct VerifyArgs {
  const char* target; int64_t tb, tp;        // bytes from sequence to sequence, from position to position
  const char* draft; int64_t db, dp;         // null: no draft distribution
  const int32_t* tokens; const int32_t* n_draft; const float* u_accept; const float* u_sample;
  int32_t* out; int32_t* accepted; float* logprobs;
  MS* stats;                                 // [row][split] in fp32; rows: [sequence][drafts] of the target, then of the draft
  VfSum* sums;                               // [row][chunk]; rows: [sequence][drafts + 1] of the target, then [sequence][drafts] of the draft; after an acceptance in
                                             // fp32: [sequence] of the target, then of the draft, the row that was stopped at
  VfSum* parts;                              // [row][split]: a block's chunks together
  double* rest;                              // [sequence][chunk]: sums of max(p - q, 0)
  uint32_t* done;                            // [sequence]: blocks that have finished; cleared by the first kernel for the second
  int B, K, V, nchunk, nstat, nsplit, npick; // splits of a row in fp32 and in fp64, blocks a sequence in the last kernel
  float c;
  double C, C2;                              // log2(e) / tau, and the power of two not below it
  double close;                              // VF_STATS: how near, relatively, u q and p may be for fp32 sums to tell which is less
};
__device__ __forceinline__ int vf_drafts(const VerifyArgs& a, int b) {
  const int n = a.n_draft ? a.n_draft[b] : a.K;
  return n < 0 ? 0 : (n > a.K ? a.K : n);
}
// 2^(z C - E), at most about 1: 32 (z C - E) = 32 k + i + r, |r| <= 1/2: 2^k * table[i] * 2^(r/32), the last one by its series to the fourth power (off by
// 1.2e-12 at most: a cumulative sum's borders move by that).  The table's 32 doubles lie in each LDS bank once: no conflicts.  What is below 2^-1000 becomes
// that (VF_NOTHING): beside a chunk's largest term it is gone, and weights are taken less twice as much, so that a masked token has none.
constexpr double VF_NOTHING = 0x1p-1000;
struct VfExp {
  const double* table;
  double C, E;                               // both times 32
  __device__ __forceinline__ double operator()(float z) const {
    constexpr double MAGIC = 6755399441055744.0, L = 0.69314718055994530942 / 32;   // 1.5 * 2^52: the sum's low bits are the whole number
    const double y = fmax(fma((double)z, C, -E), -32000.0);
    const double t = y + MAGIC, r = y - (t - MAGIC);
    const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, t);
    double p = fma(r, L * L * L * L / 24, L * L * L / 6);
    p = fma(r, p, L * L / 2);
    p = fma(r, p, L);
    p = fma(r, p, 1.0);
    p *= table[n & 31];
    return __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, p) + ((uint64_t)((n & ~31u) << 15) << 32));   // k into the exponent
  }
};
// The whole number E of a maximum m: m C rounded up.  Beyond 2^36 a float's neighbours differ by 2^12 and more in the exponent, so that beside m all but its
// equals are nothing, but m C itself is rounded by more and more: there C is replaced by the power of two above it, which makes m C2 exact, and whole.
// vf_slope says from E which of the two it was made with.
constexpr double VF_FAR = 0x1p36;
__device__ __forceinline__ double vf_slope(const VerifyArgs& a, double e) { return fabs(e) > VF_FAR ? a.C2 : a.C; }
__device__ __forceinline__ double vf_ceil(const VerifyArgs& a, float m) {
  if (m == -INFINITY) return 0.0;
  const double e = ceil((double)m * a.C);
  return fabs(e) > VF_FAR ? (double)m * a.C2 : e;
}
// probability of logit z in a row of sum `s`; what VF_NOTHING stands for is 0
__device__ __forceinline__ double vf_prob(const double* table, const VerifyArgs& a, const VfSum& s, float z) {
  const double e = VfExp{table, 32.0 * vf_slope(a, s.e), 32.0 * s.e}(z);
  return e > 2.0 * VF_NOTHING ? e / s.s : 0.0;
}
__device__ __forceinline__ double vf_scaled(const VfSum& x, double e) { return x.e == e ? x.s : ldexp(x.s, (int)fmax(x.e - e, -4000.0)); }   // s 2^(x.e - e)
__device__ __forceinline__ VfSum vf_add(const VfSum& x, const VfSum& y) {
  const double e = fmax(x.e, y.e);
  return VfSum{e, vf_scaled(x, e) + vf_scaled(y, e)};
}
__device__ __forceinline__ bool vf_good(const VfSum& x) { return x.e > -INFINITY && x.e < INFINITY && x.s > 0.0; }
__device__ __forceinline__ double vf_logp(const VerifyArgs& a, const VfSum& s, float z) {
  return fma((double)z, vf_slope(a, s.e), -s.e) * 0.69314718055994530942 - log(s.s);   // (one rounding: z C alone is off by up to 2^-17 at 2^36)
}

// (maximum, sum) of a share of one drafted position's row
template <int DT>
__global__ __launch_bounds__(VF_T) void verify_stats_kernel(VerifyArgs a) {
  constexpr int VEC = Lg<DT>::VEC, U = 32 / VEC;
  __shared__ MS red[VF_T / 64];
  const int64_t row = blockIdx.x / (uint32_t)a.nstat, trows = (int64_t)a.B * a.K;
  const int split = (int)(blockIdx.x % (uint32_t)a.nstat);
  const int64_t of = row < trows ? row : row - trows;
  const int b = (int)(of / a.K), i = (int)(of - (int64_t)b * a.K);
  if (i >= vf_drafts(a, b)) return;
  const char* z = row < trows ? a.target + b * a.tb + i * a.tp : a.draft + b * a.db + i * a.dp;
  const int nvec = (a.V + VEC - 1) / VEC;
  const int v0 = (int)((int64_t)nvec * split / a.nstat), v1 = (int)((int64_t)nvec * (split + 1) / a.nstat);
  float m = -INFINITY, s = 0.0f;
  for (int v = v0; v < v1; v += VF_T * U) {
    Pack x[U];
    if (v + VF_T * U <= v1 && (v + VF_T * U) * VEC <= a.V) {
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = tk_load16(z + (size_t)(v + u * VF_T + (int)threadIdx.x) * 16);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) { const int at = v + u * VF_T + (int)threadIdx.x; x[u] = at < v1 ? tk_load<DT>(z, at, a.V) : tk_neg<DT>(); }
    }
    float nm = m;
#pragma unroll
    for (int u = 0; u < U; ++u) { nm = fmaxf(nm, tk_max<DT>(x[u])); tk_redecode(x[u]); }
    const ExpSum es(tk_base(nm), a.c);
    float p = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u) p += es.sum<DT>(x[u]);
    p *= es.fix;
    if (es.far) {
      p = 0.0f;
#pragma unroll 1
      for (int u = 0; u < U; ++u) { const int at = v + u * VF_T + (int)threadIdx.x; if (at < v1) p += es.exact_sum<DT>(tk_load<DT>(z, at, a.V)); }
    }
    s = s * tk_exp2((m - es.b) * a.c) + p;
    m = nm;
  }
  const MS ms = block_lse<VF_T>(m, s, a.c, red);
  if (threadIdx.x == 0) a.stats[blockIdx.x] = ms;
}

// a chunk's vectors of a lane
template <int DT> __device__ __forceinline__ void vf_chunk(Pack (&y)[VF_CHUNK / 64 / Lg<DT>::VEC], const char* row, int ch, int V) {
  constexpr int U = VF_CHUNK / 64 / Lg<DT>::VEC;
  const int lane = threadIdx.x & 63;
  if ((ch + 1) * VF_CHUNK <= V) {
#pragma unroll
    for (int u = 0; u < U; ++u) y[u] = tk_load16(row + (size_t)((ch * U + u) * 64 + lane) * 16);
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) y[u] = tk_load<DT>(row, (ch * U + u) * 64 + lane, V);
  }
}

// the fp64 sum of a wave's chunk
template <int DT> __device__ __forceinline__ VfSum vf_sum_chunk(Pack (&x)[VF_CHUNK / 64 / Lg<DT>::VEC], int ch, const VerifyArgs& a, const double* table) {
  constexpr int VEC = Lg<DT>::VEC, U = VF_CHUNK / 64 / VEC;
  float m = -INFINITY;
  uint64_t nan = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    m = fmaxf(m, tk_max<DT>(x[u]));
#pragma unroll
    for (int j = 0; j < VEC; j += 2) nan |= __ballot(__builtin_isunordered(tk_get<DT>(x[u], j), tk_get<DT>(x[u], j + 1)));
  }
  m = wave_max(m);
  const double E = vf_ceil(a, m);
  const VfExp ex = {table, 32.0 * vf_slope(a, E), 32.0 * E};
  double s = 0.0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if ((ch * U + u) * 64 * VEC >= a.V) break;   // (the same for every lane)
    tk_redecode(x[u]);
#pragma unroll
    for (int j = 0; j < VEC; ++j) s += ex(tk_get<DT>(x[u], j));
  }
  s = wave_sum(s);
  if (m == -INFINITY) s = 0.0;
  if (nan) s = NAN;
  return VfSum{m == -INFINITY ? -INFINITY : E, s};
}

// the fp64 sum of a whole row, by the block's waves; every thread gets it.  `part` holds one a wave
template <int DT> __device__ VfSum vf_sum_row(const VerifyArgs& a, const char* row, const double* table, VfSum* part) {
  constexpr int U = VF_CHUNK / 64 / Lg<DT>::VEC;
  const int wave = threadIdx.x >> 6;
  VfSum all = {-INFINITY, 0.0};
  for (int ch = wave; ch < a.nchunk; ch += VF_WAVES) {
    Pack x[U];
    vf_chunk<DT>(x, row, ch, a.V);
    all = vf_add(all, vf_sum_chunk<DT>(x, ch, a, table));
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[wave] = all;
  __syncthreads();
  all = part[0];
#pragma unroll
  for (int w = 1; w < VF_WAVES; ++w) all = vf_add(all, part[w]);
  return all;
}

// How many drafts of sequence b are accepted; every thread of the block gets it.  srow: the rows' sums, target 0 .. n, draft 0 .. n - 1 behind them
// (from fp32 statistics target 0 .. n - 1; VF_ONE: the caller has filled them in).  `write`: the block that writes what is known then.
// From fp32 statistics a draft whose two sides lie nearer to each other than those can tell (a.close) is decided by fp64 sums of its rows, which each block of the
// sequence forms for itself: a few drafts in 10^5.  So a decision does not go by how many others are in the call.
enum : uint8_t { VF_NO, VF_YES, VF_CLOSE };
template <int DT, int HOW> __device__ int vf_accept(const VerifyArgs& a, int b, int n, bool write, const double* table, VfSum* srow, int* sat, uint8_t* sstate = nullptr,
                                                    VfSum* spart = nullptr) {   // (the last two: VF_STATS)
  const int tid = threadIdx.x;
  const int64_t k0 = (int64_t)b * a.K, t0 = (int64_t)b * (a.K + 1);
  int x = -1;
  float u = 0.0f, zp = 0.0f, zq = 0.0f;
  if (tid < n) {
    x = a.tokens[k0 + tid];
    u = a.u_accept[k0 + tid];
    if ((uint32_t)x < (uint32_t)a.V) {
      zp = tk_at<DT>(a.target + b * a.tb + tid * a.tp, x);
      if (a.draft) zq = tk_at<DT>(a.draft + b * a.db + tid * a.dp, x);
    }
  }
  if (tid == 0) *sat = n;
  const int heads = HOW == VF_STATS ? n : n + 1, rows = HOW == VF_ONE ? 0 : heads + (a.draft ? n : 0);
  for (int r = tid >> 4; r < rows; r += VF_T / 16) {   // 16 lanes a row
    VfSum s = {-INFINITY, 0.0};
    if constexpr (HOW == VF_SUMS) {
      const VfSum* p = a.parts + (r < heads ? t0 + r : (int64_t)a.B * (a.K + 1) + k0 + r - heads) * a.nsplit;
      for (int i = tid & 15; i < a.nsplit; i += 16) s = vf_add(s, p[i]);
      for (int o = 8; o > 0; o >>= 1) s = vf_add(s, VfSum{__shfl_xor(s.e, o, 16), __shfl_xor(s.s, o, 16)});
    } else {
      const MS* p = a.stats + (r < heads ? k0 + r : (int64_t)a.B * a.K + k0 + r - heads) * a.nstat;
      float m = -INFINITY;
      for (int i = tid & 15; i < a.nstat; i += 16) m = fmaxf(m, p[i].m);
      for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 16));
      for (int i = tid & 15; i < a.nstat; i += 16) s.s += p[i].s * (double)tk_exp2((p[i].m - tk_base(m)) * a.c);
      for (int o = 8; o > 0; o >>= 1) s.s += __shfl_xor(s.s, o, 16);
      s.e = m == -INFINITY ? m : vf_ceil(a, m);
      if ((tid & 15) == 0) s.s *= exp2(fma((double)m, vf_slope(a, s.e), -s.e));   // (the sum was relative to m)
    }
    if ((tid & 15) == 0) srow[r] = s;
  }
  __syncthreads();
  const auto decide = [&](const VfSum& ps, const VfSum& qs, double* p, double* uq) {   // thread `tid`'s draft; a row that is no distribution: not accepted
    if ((uint32_t)x >= (uint32_t)a.V || !vf_good(ps) || (a.draft && !vf_good(qs))) return false;
    *p = vf_prob(table, a, ps, zp);
    *uq = (double)u * (a.draft ? vf_prob(table, a, qs, zq) : 1.0);
    return *uq < *p;                         // (a NaN: not accepted)
  };
  double logp = 0.0;
  if (tid < n) {
    double p = 0.0, uq = 0.0;
    const bool ok = decide(srow[tid], a.draft ? srow[heads + tid] : srow[tid], &p, &uq);
    if constexpr (HOW == VF_STATS) sstate[tid] = fabs(uq - p) < a.close * fmax(uq, p) ? VF_CLOSE : (ok ? VF_YES : VF_NO);
    if (!ok || (HOW == VF_STATS && sstate[tid] == VF_CLOSE)) atomicMin(sat, tid);
    else if (HOW != VF_STATS && write) logp = vf_logp(a, srow[tid], zp);   // (before the barrier: it is on the way to the token there)
  }
  __syncthreads();
  int at = *sat;
  if constexpr (HOW == VF_STATS) {
    while (at < n && sstate[at] == VF_CLOSE) {   // (the same for every thread)
      const VfSum ps = vf_sum_row<DT>(a, a.target + b * a.tb + at * a.tp, table, spart);
      const VfSum qs = a.draft ? vf_sum_row<DT>(a, a.draft + b * a.db + at * a.dp, table, spart) : ps;
      if (tid == at) {
        double p, uq;
        sstate[at] = decide(ps, qs, &p, &uq) ? VF_YES : VF_NO;
        srow[at] = ps;
      }
      __syncthreads();
      while (at < n && sstate[at] == VF_YES) ++at;
      __syncthreads();
    }
  }
  if (write) {
    if (HOW == VF_STATS && tid < at) logp = vf_logp(a, srow[tid], zp);
    if (tid < at) { a.out[t0 + tid] = x; if (a.logprobs) a.logprobs[t0 + tid] = (float)logp; }
    else if (tid > at && tid <= a.K) { a.out[t0 + tid] = -1; if (a.logprobs) a.logprobs[t0 + tid] = 0.0f; }
    if (tid == 0) a.accepted[b] = at;
  }
  return at;
}

template <int DT, int HOW>
__global__ __launch_bounds__(VF_T) void verify_sums_kernel(VerifyArgs a) {
  constexpr int U = VF_CHUNK / 64 / Lg<DT>::VEC;
  __shared__ double table[32];
  __shared__ VfSum part[VF_WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / (uint32_t)a.nsplit;
  const int split = (int)(blockIdx.x % (uint32_t)a.nsplit);
  const char* z;
  if (tid < 32) table[tid] = exp2(tid / 32.0);
  if constexpr (HOW == VF_SUMS) {
    const int64_t trows = (int64_t)a.B * (a.K + 1);
    if (row < trows) {
      const int b = (int)(row / (a.K + 1)), i = (int)(row - (int64_t)b * (a.K + 1));
      if (i == 0 && split == 0 && tid == 0) a.done[b] = 0;
      if (i > vf_drafts(a, b)) return;
      z = a.target + b * a.tb + i * a.tp;
    } else {
      const int b = (int)((row - trows) / a.K), i = (int)(row - trows - (int64_t)b * a.K);
      if (i >= vf_drafts(a, b)) return;
      z = a.draft + b * a.db + i * a.dp;
    }
  } else {
    __shared__ VfSum srow[2 * TK_MAX_DRAFTS];
    __shared__ int sat;
    __shared__ uint8_t sstate[TK_MAX_DRAFTS];
    const bool of_draft = row >= a.B;
    const int b = (int)(of_draft ? row - a.B : row), n = vf_drafts(a, b);
    const int at = vf_accept<DT, VF_STATS>(a, b, n, !of_draft && split == 0, table, srow, &sat, sstate, part);
    if (!of_draft && split == 0 && tid == 0) a.done[b] = 0;
    if (of_draft && at >= n) return;
    z = of_draft ? a.draft + b * a.db + at * a.dp : a.target + b * a.tb + at * a.tp;
  }
  const int c0 = (int)((int64_t)a.nchunk * split / a.nsplit), c1 = (int)((int64_t)a.nchunk * (split + 1) / a.nsplit);
  Pack y[U];
  if (c0 + wave < c1) vf_chunk<DT>(y, z, c0 + wave, a.V);
  __syncthreads();
  VfSum all = {-INFINITY, 0.0};
  for (int ch = c0 + wave; ch < c1; ch += VF_WAVES) {
    Pack x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = y[u];
    if (ch + VF_WAVES < c1) vf_chunk<DT>(y, z, ch + VF_WAVES, a.V);
    const VfSum mine = vf_sum_chunk<DT>(x, ch, a, table);
    if (lane == 0) a.sums[row * a.nchunk + ch] = mine;
    all = vf_add(all, mine);
  }
  if (lane == 0) part[wave] = all;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < VF_WAVES; ++w) all = vf_add(all, part[w]);
    a.parts[row * a.nsplit + split] = all;
  }
}

// inclusive sum over the block's threads, and the whole; `ss` holds one number a wave
__device__ double vf_scan(double v, double* ss, double* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int d = 1; d < 64; d <<= 1) { const double o = __shfl_up(v, d, 64); if (lane >= d) v += o; }
  __syncthreads();
  if (lane == 63) ss[wave] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int w = 0; w < VF_WAVES; ++w) { if (w == wave) v += t; t += ss[w]; }
  *total = t;
  return v;
}

// What a token weighs in the draw: p, max(p - q, 0) where there is a draft row, or p but for one token.  p and q are known to 2.7e-12 of themselves each
// (VfExp's series, in the exponential and in the sum): what they differ by less than 2^-37 of is no difference.  Without that, of rows that are equal, or equal
// up to a constant, p - q left roundings at half of the tokens, and the token was drawn from those instead of from p.  It goes into q's factor: no work.
constexpr double VF_SAME = 0x1p-37;
template <int DT> struct VfWeight {
  const char *prow, *qrow;
  VfExp ep, eq;
  double np, nq, none;
  int V, skip;
  __device__ __forceinline__ VfWeight(const VerifyArgs& a, const double* table, const char* prow, const VfSum& ps, const char* qrow, const VfSum& qs)
    : prow(prow), qrow(qrow), ep{table, 32.0 * vf_slope(a, ps.e), 32.0 * ps.e}, eq{table, 32.0 * vf_slope(a, qs.e), 32.0 * qs.e}, np(1.0 / ps.s), nq(1.0 / qs.s * (1.0 + VF_SAME)),
      none(2.0 * VF_NOTHING * np), V(a.V), skip(-1) {}
  __device__ __forceinline__ void leave_out(int token) { if ((uint32_t)token < (uint32_t)V) skip = token; }   // a looked-up token that was rejected
  __device__ __forceinline__ bool less() const { return qrow || skip >= 0; }
  __device__ __forceinline__ void p_itself() { qrow = nullptr; skip = -1; }
  __device__ __forceinline__ double rest(float zp, float zq) const { return fmax(fma(ep(zp), np, fma(eq(zq), -nq, -none)), 0.0); }
  __device__ __forceinline__ double operator()(int e) const {
    if (e >= V || e == skip) return 0.0;
    const float zp = tk_at<DT>(prow, e);
    return qrow ? rest(zp, tk_at<DT>(qrow, e)) : fmax(fma(ep(zp), np, -none), 0.0);
  }
};

// Draws a token among the chunk from token c0 on, `below` of the weight lying before it: the first whose cumulative weight exceeds `goal` (negative: the
// chunk is all there is, the goal goes by its weight; false if it has none and could have more); rounding, or u >= 1, may leave none: the last of any weight.
template <int DT> __device__ bool vf_token(const VerifyArgs& a, int64_t o, const VfWeight<DT>& weight, const VfSum& ps, const char* prow, int c0, double below, double goal,
                                           double* ss, int* sfirst, int* slast) {
  constexpr int PER = VF_CHUNK / VF_T;
  const int e0 = c0 + threadIdx.x * PER;
  double t[PER], s = 0.0, sum;
#pragma unroll
  for (int j = 0; j < PER; ++j) { t[j] = weight(e0 + j); s += t[j]; }
  double c = below + (vf_scan(s, ss, &sum) - s);
  if (goal < 0.0) {
    if (!(sum > 0.0) && weight.less()) return false;
    const float u = a.u_sample[o / (a.K + 1)];
    goal = (u > 0.0f ? (double)u : 0.0) * sum;
  }
  if (threadIdx.x == 0) { *sfirst = a.V; *slast = -1; }
  __syncthreads();
  int first = a.V, last = -1;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    c += t[j];
    if (t[j] > 0.0) { last = e0 + j; if (c > goal && first == a.V) first = last; }
  }
  if (first < a.V) atomicMin(sfirst, first);
  if (last >= 0) atomicMax(slast, last);
  __syncthreads();
  if (threadIdx.x == 0) {
    const int token = *sfirst < a.V ? *sfirst : *slast;
    a.out[o] = token;
    if (a.logprobs) a.logprobs[o] = (float)vf_logp(a, ps, tk_at<DT>(prow, token));
  }
  return true;
}

template <int DT, int HOW>
__global__ __launch_bounds__(VF_T) void verify_pick_kernel(VerifyArgs a) {
  constexpr int VEC = Lg<DT>::VEC, U = VF_CHUNK / 64 / VEC;
  __shared__ double table[32];
  __shared__ double ss[VF_WAVES];
  __shared__ VfSum srow[HOW == VF_STATS ? 2 : 2 * TK_MAX_DRAFTS + 1];
  __shared__ int sat, sfirst, slast, slastblock;
  __shared__ double sbelow;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = (int)(blockIdx.x / (uint32_t)a.npick), part = (int)(blockIdx.x % (uint32_t)a.npick);
  const int n = vf_drafts(a, b);
  if (tid < 32) table[tid] = exp2(tid / 32.0);
  int at, prow_at, qrow_at;                  // drafts accepted; where srow holds the row that the token is drawn from, and the draft's
  int64_t prow_id;                           // which row of `sums` it is
  if constexpr (HOW == VF_SUMS) {
    at = vf_accept<DT, VF_SUMS>(a, b, n, part == 0, table, srow, &sat);
    prow_at = at; qrow_at = n + 1 + at;
    prow_id = (int64_t)b * (a.K + 1) + at;
  } else {
    at = a.accepted[b];
    prow_at = 0; qrow_at = 1;
    prow_id = b;
    if (tid < 32 && (tid < 16 || (a.draft && at < n))) {
      const VfSum* p = a.parts + (int64_t)(tid < 16 ? b : a.B + b) * a.nsplit;
      VfSum s = {-INFINITY, 0.0};
      for (int i = tid & 15; i < a.nsplit; i += 16) s = vf_add(s, p[i]);
      for (int o = 8; o > 0; o >>= 1) s = vf_add(s, VfSum{__shfl_xor(s.e, o, 16), __shfl_xor(s.s, o, 16)});
      if ((tid & 15) == 0) srow[tid >> 4] = s;
    }
    __syncthreads();
  }
  const int64_t o = (int64_t)b * (a.K + 1) + at;
  const VfSum ps = srow[prow_at];
  if (!vf_good(ps)) {                        // no distribution to draw from
    if (part == 0 && tid == 0) { a.out[o] = -1; if (a.logprobs) a.logprobs[o] = 0.0f; }
    return;
  }
  const char* prow = a.target + b * a.tb + at * a.tp;
  const char* qrow = a.draft && at < n && vf_good(srow[qrow_at]) ? a.draft + b * a.db + at * a.dp : nullptr;
  const VfSum qs = qrow ? srow[qrow_at] : VfSum{0.0, 1.0};
  VfWeight<DT> weight(a, table, prow, ps, qrow, qs);
  if (qrow) {
    for (int ch = part * VF_WAVES + wave; ch < a.nchunk; ch += a.npick * VF_WAVES) {
      Pack px[U], qx[U];
      vf_chunk<DT>(px, prow, ch, a.V);
      vf_chunk<DT>(qx, qrow, ch, a.V);
      double s = 0.0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if ((ch * U + u) * 64 * VEC >= a.V) break;
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += weight.rest(tk_get<DT>(px[u], j), tk_get<DT>(qx[u], j));
      }
      s = wave_sum(s);
      if (lane == 0) __hip_atomic_store(&a.rest[(int64_t)b * a.nchunk + ch], s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (a.npick > 1) {                       // the last block to come by sees what all have written: the sums are written through and read past the caches
                                             // (agent scope), each wave waits for its own, then the block counts; a whole-cache write-back per block cost 100 us
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (tid == 0) slastblock = __hip_atomic_fetch_add(&a.done[b], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)a.npick - 1;
      __syncthreads();
      if (!slastblock) return;
    } else __syncthreads();
  } else if (part != 0) return;

  // the chunk that the goal falls into; a thread looks at neighbouring chunks
  if (!a.draft && at < n) weight.leave_out(a.tokens[(int64_t)b * a.K + at]);
  const VfSum* sums = a.sums + prow_id * a.nchunk;
  const int per = (a.nchunk + VF_T - 1) / VF_T;
  const float u = a.u_sample[b];
  double total, goal, before;
  for (;;) {
    double without = 0.0;                    // the skipped token's chunk, summed again without it
    const int skip = weight.skip;
    if (skip >= 0) {
      double w = 0.0;
      for (int j = 0; j < VF_CHUNK / VF_T; ++j) w += weight(skip / VF_CHUNK * VF_CHUNK + tid * (VF_CHUNK / VF_T) + j);
      (void)vf_scan(w, ss, &without);
    }
    const auto chunk = [&](int i) {
      if (i >= a.nchunk) return 0.0;
      if (weight.qrow) return (double)__hip_atomic_load(&a.rest[(int64_t)b * a.nchunk + i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (skip >= 0 && i == skip / VF_CHUNK) return without;
      // a chunk that counts has a token that counts: its largest is above 2^-991 of the row's, and weight() leaves out what is below 2^-999
      return sums[i].e - ps.e >= -990.0 ? vf_scaled(sums[i], ps.e) * weight.np : 0.0;
    };
    double mine = 0.0;
    for (int j = 0; j < per; ++j) mine += chunk(tid * per + j);
    before = vf_scan(mine, ss, &total) - mine;
    if (!(total > 0.0) && weight.less()) { weight.p_itself(); continue; }   // nothing left of p
    if (tid == 0) { sfirst = a.nchunk; slast = -1; }
    __syncthreads();
    goal = (u > 0.0f ? (double)u : 0.0) * total;
    double c = before;
    int first = a.nchunk, last = -1;
    for (int j = 0; j < per; ++j) {
      const double w = chunk(tid * per + j);
      c += w;
      if (w > 0.0) { last = tid * per + j; if (c > goal && first == a.nchunk) first = last; }
    }
    if (first < a.nchunk) atomicMin(&sfirst, first);
    if (last >= 0) atomicMax(&slast, last);
    __syncthreads();
    const int hit = sfirst < a.nchunk ? sfirst : slast;   // (rounding, or u >= 1, may leave no sum above the goal: the last weight there is)
    if (hit / per == tid) { c = before; for (int j = tid * per; j < hit; ++j) c += chunk(j); sbelow = c; }
    __syncthreads();
    vf_token<DT>(a, o, weight, ps, prow, hit * VF_CHUNK, sbelow, goal, ss, &sfirst, &slast);
    break;
  }
}

// Rows of one chunk and few of them: a block a sequence.  Up to 16 lanes' vectors: 16 rows at once, else a wave a row.  The weights of the row that is
// drawn from are looked at once.  Held to 128 registers (4 waves a SIMD), at which 34 (fp32) or 4 (16 bits) are spilled to scratch, 140 and 20 bytes a lane.
template <int DT>
__global__ __launch_bounds__(VF_T, 4) void verify_one_kernel(VerifyArgs a) {
  constexpr int VEC = Lg<DT>::VEC, U = VF_CHUNK / 64 / VEC;
  __shared__ double table[32];
  __shared__ double ss[VF_WAVES];
  __shared__ VfSum srow[2 * TK_MAX_DRAFTS + 1];
  __shared__ int sat, sfirst, slast;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = (int)blockIdx.x, n = vf_drafts(a, b), rows = n + 1 + (a.draft ? n : 0);
  const auto at_row = [&](int r) { return r <= n ? a.target + b * a.tb + r * a.tp : a.draft + b * a.db + (r - n - 1) * a.dp; };
  if (tid < 32) table[tid] = exp2(tid / 32.0);
  __syncthreads();
  if (a.V <= 16 * VEC) {
    for (int r = tid >> 4; r < rows; r += VF_T / 16) {
      const Pack x = tk_load<DT>(at_row(r), tid & 15, a.V);
      float m = tk_max<DT>(x);
      bool nan = false;
#pragma unroll
      for (int j = 0; j < VEC; j += 2) nan |= __builtin_isunordered(tk_get<DT>(x, j), tk_get<DT>(x, j + 1));
      for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 16));
      const double E = vf_ceil(a, m);
      const VfExp ex = {table, 32.0 * vf_slope(a, E), 32.0 * E};
      double s = 0.0;
#pragma unroll
      for (int j = 0; j < VEC; ++j) s += ex(tk_get<DT>(x, j));
      if (m == -INFINITY) s = 0.0;
      if (nan) s = NAN;
      for (int o = 8; o > 0; o >>= 1) s += __shfl_xor(s, o, 16);
      if ((tid & 15) == 0) srow[r] = VfSum{m == -INFINITY ? -INFINITY : E, s};
    }
  } else {
    Pack y[U];
    if (wave < rows) vf_chunk<DT>(y, at_row(wave), 0, a.V);
    for (int r = wave; r < rows; r += VF_WAVES) {
      Pack x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = y[u];
      if (r + VF_WAVES < rows) vf_chunk<DT>(y, at_row(r + VF_WAVES), 0, a.V);
      const VfSum sum = vf_sum_chunk<DT>(x, 0, a, table);
      if (lane == 0) srow[r] = sum;
    }
  }
  const int at = vf_accept<DT, VF_ONE>(a, b, n, true, table, srow, &sat);
  const int64_t o = (int64_t)b * (a.K + 1) + at;
  const VfSum ps = srow[at];
  if (!vf_good(ps)) {
    if (tid == 0) { a.out[o] = -1; if (a.logprobs) a.logprobs[o] = 0.0f; }
    return;
  }
  const bool less = a.draft && at < n && vf_good(srow[n + 1 + at]);
  VfWeight<DT> weight(a, table, at_row(at), ps, less ? at_row(n + 1 + at) : nullptr, less ? srow[n + 1 + at] : VfSum{0.0, 1.0});
  if (!a.draft && at < n) weight.leave_out(a.tokens[(int64_t)b * a.K + at]);
  while (!vf_token<DT>(a, o, weight, ps, at_row(at), 0, 0.0, -1.0, ss, &sfirst, &slast)) weight.p_itself();
}

// tau = 0: p is one-hot at the row's largest logit (the lowest index of equal ones), a draft is accepted where it is that token
struct VfBest { float m; int32_t idx, bad, pad; };   // bad: a NaN or +inf among the logits
__device__ __forceinline__ void vf_better(float& m, int& idx, float om, int oi) { if (om > m || (om == m && oi < idx)) { m = om; idx = oi; } }

template <int DT>
__global__ __launch_bounds__(VF_T) void verify_best_kernel(VerifyArgs a) {
  constexpr int VEC = Lg<DT>::VEC, U = 4;
  __shared__ VfBest red[VF_T / 64];
  uint32_t id = blockIdx.x;
  const int split = (int)(id % (uint32_t)a.nsplit); id /= (uint32_t)a.nsplit;
  const int b = (int)(id % (uint32_t)a.B), i = (int)(id / (uint32_t)a.B), tid = threadIdx.x;
  if (i > vf_drafts(a, b)) return;
  const char* row = a.target + b * a.tb + i * a.tp;
  const int nvec = (a.V + VEC - 1) / VEC;
  const int v0 = (int)((int64_t)nvec * split / a.nsplit), v1 = (int)((int64_t)nvec * (split + 1) / a.nsplit);
  float m = -INFINITY;
  int idx = a.V, bad = 0;
  for (int v = v0; v < v1; v += VF_T * U) {
    Pack x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) { const int at = v + u * VF_T + tid; x[u] = at < v1 ? tk_load<DT>(row, at, a.V) : tk_neg<DT>(); }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float z = tk_get<DT>(x[u], j);
        if (z > m) { m = z; idx = (v + u * VF_T + tid) * VEC + j; }
        bad |= !(z < INFINITY);
      }
  }
  for (int o = 32; o > 0; o >>= 1) {
    const float om = __shfl_xor(m, o, 64);
    const int oi = __shfl_xor(idx, o, 64);
    bad |= __shfl_xor(bad, o, 64);
    vf_better(m, idx, om, oi);
  }
  if ((tid & 63) == 0) red[tid >> 6] = VfBest{m, idx, bad, 0};
  __syncthreads();
  if (tid == 0) {
    for (int k = 1; k < VF_T / 64; ++k) { vf_better(m, idx, red[k].m, red[k].idx); bad |= red[k].bad; }
    reinterpret_cast<VfBest*>(a.sums)[blockIdx.x] = VfBest{m, idx, bad, 0};
  }
}
__global__ __launch_bounds__(VF_T) void verify_greedy_kernel(VerifyArgs a) {
  __shared__ int sa;
  const int tid = threadIdx.x, b = blockIdx.x, n = vf_drafts(a, b);
  if (tid == 0) sa = n;
  __syncthreads();
  int best = -1;
  if (tid <= n) {
    const VfBest* st = reinterpret_cast<const VfBest*>(a.sums) + ((int64_t)tid * a.B + b) * a.nsplit;
    float m = -INFINITY;
    int idx = a.V, bad = 0;
    for (int k = 0; k < a.nsplit; ++k) { vf_better(m, idx, st[k].m, st[k].idx); bad |= st[k].bad; }
    if (!bad && m > -INFINITY) best = idx;
  }
  if (tid < n && (best < 0 || a.tokens[(int64_t)b * a.K + tid] != best)) atomicMin(&sa, tid);
  __syncthreads();
  if (tid <= a.K) {
    a.out[(int64_t)b * (a.K + 1) + tid] = tid <= sa ? best : -1;
    if (a.logprobs) a.logprobs[(int64_t)b * (a.K + 1) + tid] = 0.0f;
  }
  if (tid == 0) a.accepted[b] = sa;
}

struct VerifyPlan { int how, nchunk, nstat, nsplit, npick; size_t o_parts, o_rest, o_stats, o_done, ws; };
VerifyPlan verify_plan(int dtype, int B, int K, int V, bool draft, bool greedy) {
  VerifyPlan p = {};
  p.nchunk = (V + VF_CHUNK - 1) / VF_CHUNK;
  // One kernel saves a launch, the workspace and the blocks' own acceptance, but has four waves for all rows of a sequence: us of the GPU, one / two kernels,
  // fp32 with draft logits: 18 tokens: 120 sequences of 7 drafts 8 / 19, 1000 of 128 31 / 854, one of 128 20 / 26;  300 tokens: one sequence of 3 drafts
  // 12 / 17, of 16 25 / 19, 120 of 16 26 / 30, of 40 46 / 49;  2048 tokens: one of 3 17 / 17, of 7 21 / 17, 120 of 16 37 / 37, of 40 67 / 50, 1000 of 128 496 / 634
  const int own = K + 1 + (draft ? K : 0);
  if (!greedy && p.nchunk == 1 && (V <= 16 * (dtype == CBM_F32 ? 4 : 8) || own <= 12 || 3 * own <= B)) { p.how = VF_ONE; return p; }
  const int64_t all = (int64_t)B * (K + 1) + (draft && !greedy ? (int64_t)B * K : 0);
  // fp64 sums of every row up to 2^24 logits (about 12 us of fp64 beside a launch saved of 5); beyond, of the rows that tokens are drawn from
  p.how = greedy || K == 0 || all * V <= (1 << 24) ? VF_SUMS : VF_STATS;
  const int64_t rows = p.how == VF_SUMS ? all : (int64_t)B * (draft ? 2 : 1);
  const int most = (p.nchunk + VF_WAVES - 1) / VF_WAVES;   // a chunk a wave
  // blocks: about 16384 of the fp64 sums, 1024 in the last kernel, 8192 of the fp32 statistics
  const auto share = [](int64_t blocks, int64_t of, int most) { const int64_t n = (blocks + of - 1) / of; return (int)(n < most ? n : most); };
  p.nsplit = share(16384, rows, most);
  p.npick = draft && K > 0 ? share(1024, B, most) : 1;
  p.nstat = p.how == VF_SUMS ? 0 : share(8192, all, (V + 8191) / 8192);
  if (greedy) { p.ws = (size_t)rows * p.nsplit * sizeof(VfBest); return p; }
  p.o_parts = (size_t)rows * p.nchunk * sizeof(VfSum);
  p.o_rest = p.o_parts + (size_t)rows * p.nsplit * sizeof(VfSum);
  p.o_stats = p.o_rest + (size_t)B * p.nchunk * sizeof(double);
  p.o_done = p.o_stats + (size_t)B * K * (draft ? 2 : 1) * p.nstat * sizeof(MS);
  p.ws = p.o_done + (size_t)B * sizeof(uint32_t);
  return p;
}
template <int DT> void verify_dispatch(const VerifyArgs& a, const VerifyPlan& p, bool greedy, hipStream_t st) {
  if (greedy) {
    hipLaunchKernelGGL(verify_best_kernel<DT>, dim3((uint32_t)((int64_t)a.B * (a.K + 1) * a.nsplit)), dim3(VF_T), 0, st, a);
    hipLaunchKernelGGL(verify_greedy_kernel, dim3(a.B), dim3(VF_T), 0, st, a);
    return;
  }
  if (p.how == VF_ONE) {
    hipLaunchKernelGGL(verify_one_kernel<DT>, dim3(a.B), dim3(VF_T), 0, st, a);
  } else if (p.how == VF_SUMS) {
    const int64_t rows = (int64_t)a.B * (a.K + 1) + (a.draft ? (int64_t)a.B * a.K : 0);
    hipLaunchKernelGGL((verify_sums_kernel<DT, VF_SUMS>), dim3((uint32_t)(rows * a.nsplit)), dim3(VF_T), 0, st, a);
    hipLaunchKernelGGL((verify_pick_kernel<DT, VF_SUMS>), dim3((uint32_t)a.B * a.npick), dim3(VF_T), 0, st, a);
  } else {
    const int64_t rows = (int64_t)a.B * (a.draft ? 2 : 1);
    hipLaunchKernelGGL(verify_stats_kernel<DT>, dim3((uint32_t)(rows * a.K * a.nstat)), dim3(VF_T), 0, st, a);
    hipLaunchKernelGGL((verify_sums_kernel<DT, VF_STATS>), dim3((uint32_t)(rows * a.nsplit)), dim3(VF_T), 0, st, a);
    hipLaunchKernelGGL((verify_pick_kernel<DT, VF_STATS>), dim3((uint32_t)a.B * a.npick), dim3(VF_T), 0, st, a);
  }
}

// ------------------------------------------------------------------------------------------ entry points: checks, plan, launches
#define TK_REFUSE(...) do { cbm_set_error(__VA_ARGS__); return -1; } while (0)
bool tk_temperature(double t) { return t >= 1e-4 && t <= 1e4; }
int tk_es(int dtype) { return dtype == CBM_F32 ? 4 : 2; }
int tk_rows(const char* fn, int dtype, int64_t rows, int vocab) {
  if (dtype != CBM_F32 && dtype != CBM_BF16 && dtype != CBM_F16) TK_REFUSE("%s: dtype %d is none of CBM_F32, CBM_BF16, CBM_F16", fn, dtype);
  if (vocab < 1 || vocab > TK_MAX_VOCAB) TK_REFUSE("%s: vocab %d outside [1, %d]", fn, vocab, TK_MAX_VOCAB);
  if (rows < 0 || rows >= TK_MAX_ROWS) TK_REFUSE("%s: %lld rows outside [0, 2^22)", fn, (long long)rows);
  return 0;
}
int tk_pointer(const char* fn, const char* name, const void* p, size_t align) {
  if (!p) TK_REFUSE("%s: %s is null", fn, name);
  if ((uintptr_t)p % align) TK_REFUSE("%s: %s is not aligned to its %zu-byte elements", fn, name, align);
  return 0;
}
int tk_workspace(const char* fn, const void* ws, int64_t have, size_t need) {
  if (need == 0) return 0;
  if (have < (int64_t)need) TK_REFUSE("%s: the workspace holds %lld bytes, %zu are needed", fn, (long long)have, need);
  return tk_pointer(fn, "workspace", ws, 16);
}
// the context's device for the time of a call, the caller's afterwards
struct DeviceScope {
  int before = -1;
  bool ok = false;
  explicit DeviceScope(const cbm_ctx* c) {
    if (hipGetDevice(&before) != hipSuccess) { before = -1; return; }
    ok = before == c->cfg.device || hipSetDevice(c->cfg.device) == hipSuccess;
    if (before == c->cfg.device) before = -1;
  }
  ~DeviceScope() { if (before >= 0) (void)hipSetDevice(before); }
};
int tk_done(const char* fn) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) TK_REFUSE("%s: launch failed: %s", fn, hipGetErrorString(e));
  return 0;
}
hipStream_t tk_stream(cbm_ctx* c, void* stream) { return stream == CBM_LEARNER_STREAM ? c->lstream : (hipStream_t)stream; }
constexpr double TK_LOG2E = 1.4426950408889634074;

}  // namespace

extern "C" int64_t cbm_top_logits_workspace(int32_t dtype, int32_t rows, int32_t vocab, int32_t k) {
  if (tk_rows("cbm_top_logits_workspace", dtype, rows, vocab)) return -1;
  if (k < 1 || k > TK_MAX_TOP) TK_REFUSE("cbm_top_logits_workspace: k %d outside [1, %d]", k, TK_MAX_TOP);
  return rows ? (int64_t)top_plan(rows, vocab, k).ws : 0;
}
extern "C" int cbm_top_logits(cbm_ctx* c, const void* logits, int32_t dtype, int32_t rows, int32_t vocab, int64_t row_stride, int32_t k,
                              double temperature, int32_t* idx, float* values, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* fn = "cbm_top_logits";
  if (tk_rows(fn, dtype, rows, vocab)) return -1;
  if (k < 1 || k > TK_MAX_TOP) TK_REFUSE("%s: k %d outside [1, %d]", fn, k, TK_MAX_TOP);
  if (!tk_temperature(temperature)) TK_REFUSE("%s: temperature %g outside [1e-4, 1e4]", fn, temperature);
  if (rows > 1 && row_stride < vocab) TK_REFUSE("%s: row stride %lld is smaller than the vocabulary %d", fn, (long long)row_stride, vocab);
  if (rows == 0) { if (!c) TK_REFUSE("%s: null context", fn); return 0; }
  const int es = tk_es(dtype);
  if (tk_pointer(fn, "logits", logits, es) || tk_pointer(fn, "idx", idx, 4) || tk_pointer(fn, "values", values, 4) || tk_pointer(fn, "lse", lse, 4)) return -1;
  const TopPlan p = top_plan(rows, vocab, k);
  if (tk_workspace(fn, workspace, workspace_bytes, p.ws)) return -1;
  if (!c) TK_REFUSE("%s: null context", fn);
  DeviceScope dev(c);
  if (!dev.ok) TK_REFUSE("%s: cannot select device %d", fn, c->cfg.device);
  TopArgs a = {};
  a.logits = (const char*)logits; a.ld = row_stride * es;
  a.idx = idx; a.val = values; a.lse = lse;
  a.ws_keys = (uint64_t*)workspace; a.ws_ms = (MS*)((char*)workspace + (size_t)rows * p.nsplit * k * 8);
  a.V = vocab; a.K = k; a.rows = rows; a.nsplit = p.nsplit; a.cap = p.cap;
  a.inv_tau = 1.0 / temperature; a.c = (float)(TK_LOG2E * a.inv_tau);
  hipStream_t st = tk_stream(c, stream);
  if (dtype == CBM_F32) top_dispatch<CBM_F32>(a, p, st);
  else if (dtype == CBM_BF16) top_dispatch<CBM_BF16>(a, p, st);
  else top_dispatch<CBM_F16>(a, p, st);
  return tk_done(fn);
}

extern "C" int cbm_distill_loss_grad(cbm_ctx* c, const void* logits, int32_t dtype, int32_t rows, int32_t vocab, int64_t row_stride,
                                     const int32_t* teacher_idx, const float* teacher_logits, int32_t k, const float* teacher_lse,
                                     const float* row_weight, double temperature, float* loss, void* dlogits, int64_t grad_stride, void* stream) {
  const char* fn = "cbm_distill_loss_grad";
  if (tk_rows(fn, dtype, rows, vocab)) return -1;
  if (k < 1 || k > TK_MAX_TOP) TK_REFUSE("%s: k %d outside [1, %d]", fn, k, TK_MAX_TOP);
  if (!tk_temperature(temperature)) TK_REFUSE("%s: temperature %g outside [1e-4, 1e4]", fn, temperature);
  if (rows > 1 && row_stride < vocab) TK_REFUSE("%s: row stride %lld is smaller than the vocabulary %d", fn, (long long)row_stride, vocab);
  if (rows > 1 && dlogits && grad_stride < vocab) TK_REFUSE("%s: gradient stride %lld is smaller than the vocabulary %d", fn, (long long)grad_stride, vocab);
  if (rows == 0) { if (!c) TK_REFUSE("%s: null context", fn); return 0; }
  const int es = tk_es(dtype);
  if (tk_pointer(fn, "logits", logits, es) || tk_pointer(fn, "teacher_idx", teacher_idx, 4) || tk_pointer(fn, "teacher_logits", teacher_logits, 4) || tk_pointer(fn, "loss", loss, 4)) return -1;
  if (dlogits) {
    if (tk_pointer(fn, "dlogits", dlogits, es)) return -1;
    const uintptr_t l0 = (uintptr_t)logits, g0 = (uintptr_t)dlogits;
    const uintptr_t l1 = l0 + ((uint64_t)(rows - 1) * row_stride + vocab) * es, g1 = g0 + ((uint64_t)(rows - 1) * grad_stride + vocab) * es;
    if (l0 < g1 && g0 < l1 && !(l0 == g0 && (rows == 1 || row_stride == grad_stride)))
      TK_REFUSE("%s: dlogits overlaps logits without being the same rows (in place: the same pointer and stride)", fn);
  }
  if (!c) TK_REFUSE("%s: null context", fn);
  DeviceScope dev(c);
  if (!dev.ok) TK_REFUSE("%s: cannot select device %d", fn, c->cfg.device);
  DistillArgs a = {};
  a.logits = (const char*)logits; a.ld = row_stride * es;
  a.grad = (char*)dlogits; a.ldg = grad_stride * es;
  a.idx = teacher_idx; a.val = teacher_logits; a.lse = teacher_lse; a.weight = row_weight; a.loss = loss;
  a.rows = rows; a.V = vocab; a.K = k;
  a.tau = temperature; a.inv_tau = 1.0 / a.tau; a.c = (float)(TK_LOG2E * a.inv_tau);
  hipStream_t st = tk_stream(c, stream);
  if (dtype == CBM_F32) distill_dispatch<CBM_F32>(a, st);
  else if (dtype == CBM_BF16) distill_dispatch<CBM_BF16>(a, st);
  else distill_dispatch<CBM_F16>(a, st);
  return tk_done(fn);
}

static int verify_check(const char* fn, int dtype, int B, int K, int V, double temperature) {
  if (tk_rows(fn, dtype, B, V)) return -1;
  if (K < 0 || K > TK_MAX_DRAFTS) TK_REFUSE("%s: %d drafts outside [0, %d]", fn, K, TK_MAX_DRAFTS);
  if (!(temperature == 0.0 || tk_temperature(temperature))) TK_REFUSE("%s: temperature %g is neither 0 nor in [1e-4, 1e4]", fn, temperature);
  if ((int64_t)B * (2 * K + 1) >= TK_MAX_ROWS) TK_REFUSE("%s: %d sequences of %d drafts are 2^22 rows or more", fn, B, K);
  return 0;
}
extern "C" int64_t cbm_verify_drafts_workspace(int32_t dtype, int32_t batch, int32_t drafts, int32_t vocab, int32_t with_draft_logits, double temperature) {
  if (verify_check("cbm_verify_drafts_workspace", dtype, batch, drafts, vocab, temperature)) return -1;
  return batch ? (int64_t)verify_plan(dtype, batch, drafts, vocab, with_draft_logits != 0, temperature == 0.0).ws : 0;
}
extern "C" int cbm_verify_drafts(cbm_ctx* c, const void* target_logits, int32_t dtype, int32_t batch, int32_t drafts, int32_t vocab,
                                 int64_t target_batch_stride, int64_t target_pos_stride, const void* draft_logits, int64_t draft_batch_stride,
                                 int64_t draft_pos_stride, const int32_t* draft_tokens, const int32_t* n_draft, const float* u_accept,
                                 const float* u_sample, double temperature, int32_t* tokens, int32_t* accepted, float* logprobs, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  const char* fn = "cbm_verify_drafts";
  if (verify_check(fn, dtype, batch, drafts, vocab, temperature)) return -1;
  const bool greedy = temperature == 0.0;
  if ((drafts > 0 && target_pos_stride < 0) || (batch > 1 && target_batch_stride < 0)) TK_REFUSE("%s: negative stride", fn);
  if (draft_logits && ((drafts > 1 && draft_pos_stride < 0) || (batch > 1 && draft_batch_stride < 0))) TK_REFUSE("%s: negative stride", fn);
  if (batch == 0) { if (!c) TK_REFUSE("%s: null context", fn); return 0; }
  const int es = tk_es(dtype);
  if (tk_pointer(fn, "target_logits", target_logits, es) || tk_pointer(fn, "tokens", tokens, 4) || tk_pointer(fn, "accepted", accepted, 4)) return -1;
  if (drafts > 0 && tk_pointer(fn, "draft_tokens", draft_tokens, 4)) return -1;
  if (drafts > 0 && !greedy && tk_pointer(fn, "u_accept", u_accept, 4)) return -1;
  if (!greedy && tk_pointer(fn, "u_sample", u_sample, 4)) return -1;
  if (draft_logits && tk_pointer(fn, "draft_logits", draft_logits, es)) return -1;
  if (drafts == 0 || greedy) draft_logits = nullptr;   // (not looked at)
  const VerifyPlan p = verify_plan(dtype, batch, drafts, vocab, draft_logits != nullptr, greedy);
  if (tk_workspace(fn, workspace, workspace_bytes, p.ws)) return -1;
  if (!c) TK_REFUSE("%s: null context", fn);
  DeviceScope dev(c);
  if (!dev.ok) TK_REFUSE("%s: cannot select device %d", fn, c->cfg.device);
  VerifyArgs a = {};
  a.target = (const char*)target_logits; a.tb = target_batch_stride * es; a.tp = target_pos_stride * es;
  a.draft = (const char*)draft_logits; a.db = draft_batch_stride * es; a.dp = draft_pos_stride * es;
  a.tokens = draft_tokens; a.n_draft = n_draft; a.u_accept = u_accept; a.u_sample = u_sample;
  a.out = tokens; a.accepted = accepted; a.logprobs = logprobs;
  char* ws = (char*)workspace;
  a.sums = (VfSum*)ws; a.parts = (VfSum*)(ws + p.o_parts); a.rest = (double*)(ws + p.o_rest); a.stats = (MS*)(ws + p.o_stats); a.done = (uint32_t*)(ws + p.o_done);
  a.B = batch; a.K = drafts; a.V = vocab; a.nsplit = p.nsplit; a.nchunk = p.nchunk; a.nstat = p.nstat; a.npick = p.npick;
  // A sum in fp32 (verify_stats_kernel) is off by, in units of 2^-24: three roundings of an argument, weighted by the probabilities (3 log2 V <= 57), the exponential
  // and the join (12), the terms of a step (32), four a step (rescaling, adding).  p and q have one each.
  const int64_t step = VF_T * 32, steps = p.nstat ? ((vocab + p.nstat - 1) / p.nstat + 8 + step - 1) / step : 0;   // (a split's end is rounded to a vector)
  a.close = 2.0 * (57 + 12 + 32 + 4 * (double)steps) * 0x1p-24;
  a.C = greedy ? 0.0 : TK_LOG2E / temperature; a.C2 = greedy ? 0.0 : std::exp2(std::ceil(std::log2(a.C))); a.c = (float)a.C;
  hipStream_t st = tk_stream(c, stream);
  if (dtype == CBM_F32) verify_dispatch<CBM_F32>(a, p, greedy, st);
  else if (dtype == CBM_BF16) verify_dispatch<CBM_BF16>(a, p, greedy, st);
  else verify_dispatch<CBM_F16>(a, p, greedy, st);
  return tk_done(fn);
}

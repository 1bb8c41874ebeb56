// tokens.hip — operators of token policies: rows of logits over a whole vocabulary instead of the <= 28 actions of pointwise.hip.
//   cbm_top_logits         the K largest logits of each row, their indices, the row's log-sum-exp (what a teacher hands to its student)
//   cbm_distill_loss_grad  distillation from a teacher's top logits: loss and gradient in one call, as cbm_ppo_loss_grad / cbm_impala_loss_grad
//   cbm_verify_drafts      drafted tokens against the target's probabilities (the truncated ratio of cbm_vtrace, per token), and the next token
// All are bound by reading the logits once (the gradient: and writing it once).  Rows start at any element (odd vocabularies): 16-byte loads
// at element alignment, which the load unit takes.  Row statistics are (maximum, sum) pairs: sums of up to a few hundred terms a thread in
// fp32, everything across threads and everything that a decision or a loss depends on in fp64.
#include "cbm_ctx.h"
#include <float.h>
#include <math.h>

namespace {

constexpr int TK_MAX_VOCAB = 1 << 19;   // indices are 19 bits of a key in the top-K kernels; a row's bitmap (one bit a token) fits 64 KB of LDS
constexpr int TK_MAX_TOP = 256;         // slots of a row: four a lane of the wave that owns the row's teacher
constexpr int TK_MAX_DRAFTS = 128;      // one thread a draft in the acceptance step

// ------------------------------------------------------------------------------------------ 16 bytes of logits
struct Pack { uint32_t w[4]; };
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
__device__ __forceinline__ void tk_redecode(Pack& x) { asm volatile("" : "+v"(x.w[0]), "+v"(x.w[1]), "+v"(x.w[2]), "+v"(x.w[3])); }
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
        if constexpr (ES == 4) __builtin_memcpy(&x.w[j], row + (size_t)(e + j) * 4, 4);
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
// One block a row.  The row's first NV vectors a thread stay in registers, so that the logits are read once for statistics and gradient; what
// lies behind them is read twice.  With a tail, a bitmap of the top tokens keeps them out of the streamed sum: s_T is then a sum of its own with
// a maximum of its own, not a difference that cancels, and the top tokens join it from the wave that holds the teacher.  Every other token's
// gradient is one coefficient times exp2((z - ref) c); the top tokens' gradients are stored last, over what the stream left there.
struct DistillArgs {
  const char* logits; int64_t ld;            // bytes from row to row
  char* grad; int64_t ldg;                   // null: loss only
  const int32_t* idx; const float* val; const float* lse; const float* weight;
  float* loss;
  int V, K;
  float c;                                   // log2(e) / tau
  double inv_tau, tau;
};
template <int DT, int T, int NV, bool TAIL>
__global__ __launch_bounds__(T) void distill_kernel(DistillArgs a) {
  constexpr int VEC = Lg<DT>::VEC, ES = Lg<DT>::ES;
  __shared__ MS red[T / 64];
  __shared__ int32_t sidx[TK_MAX_TOP];
  __shared__ float sz[TK_MAX_TOP];           // the student's logits at them
  __shared__ double st[TK_MAX_TOP], slt[TK_MAX_TOP];   // t_k and log t_k
  __shared__ bool sfirst[TK_MAX_TOP];        // whether a slot is the first one of its token
  __shared__ double steacher[2];             // sum of t_k, t_T
  __shared__ MS stop;                        // TAIL: (maximum, sum) of the student's logits at the top tokens
  extern __shared__ uint32_t bits[];         // TAIL: bit j set: token j is a top token
  const int tid = threadIdx.x, V = a.V, K = a.K;
  const int64_t r = blockIdx.x;
  const char* row = a.logits + r * a.ld;
  char* grow = a.grad ? a.grad + r * a.ldg : nullptr;
  const float w = a.weight ? a.weight[r] : 1.0f;
  const int nfull = V / VEC, rem = V - nfull * VEC;

  const auto zeros = [&] {   // a row without a loss
    if (tid == 0) a.loss[r] = 0.0f;
    if (!grow) return;
    const Pack z = {{0, 0, 0, 0}};
    for (int v = tid; v < nfull; v += T) tk_store16(grow + (size_t)v * 16, z);
    if (tid < rem) tk_set<DT>(grow, nfull * VEC + tid, 0.0f);
  };
  if (w == 0.0f) return zeros();   // padding: the row is not looked at

  // the row, as far as it stays
  Pack x[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = i * T + tid;
    x[i] = v < nfull ? tk_load16(row + (size_t)v * 16) : tk_neg<DT>();
  }
  const float xe = tid < rem ? tk_at<DT>(row, nfull * VEC + tid) : -INFINITY;   // the row's last few elements, one a thread

  // the teacher's slots
  int my = -1;
  for (int k = tid; k < K; k += T) {
    my = a.idx[r * K + k];
    if ((uint32_t)my >= (uint32_t)V) my = -1;   // -1 and whatever lies outside the vocabulary: an empty slot
    sidx[k] = my;
    sz[k] = my >= 0 ? tk_at<DT>(row, my) : -INFINITY;
  }
  if constexpr (TAIL) for (int i = tid; i < (V + 31) / 32; i += T) bits[i] = 0;
  __syncthreads();
  for (int k = tid; k < K; k += T) {
    const int t = sidx[k];
    if constexpr (TAIL) if (t >= 0) atomicOr(&bits[t >> 5], 1u << (t & 31));
    bool first = t >= 0;
    for (int j = 0; j < k; ++j) first = first && sidx[j] != t;
    sfirst[k] = first;
  }
  if (tid < 64) {                             // t_k in fp64: a few exps, under the row's loads
    float v[TK_MAX_TOP / 64];
    float vm = -INFINITY;
#pragma unroll
    for (int q = 0; q < TK_MAX_TOP / 64; ++q) {
      const int k = q * 64 + tid;
      v[q] = k < K && sidx[k] >= 0 ? a.val[r * K + k] : -INFINITY;
      vm = fmaxf(vm, v[q]);
    }
    double lt[TK_MAX_TOP / 64], t[TK_MAX_TOP / 64], sum = 0.0;
    const double ref = TAIL ? (double)a.lse[r] : (double)tk_base(wave_max(vm)) * a.inv_tau;
#pragma unroll
    for (int q = 0; q < TK_MAX_TOP / 64; ++q) {
      lt[q] = (double)v[q] * a.inv_tau - ref;
      t[q] = v[q] == -INFINITY ? 0.0 : exp(lt[q]);
      sum += t[q];
    }
    sum = wave_sum(sum);
    const double logsum = TAIL || !(sum > 0.0) ? 0.0 : log(sum), scale = TAIL || !(sum > 0.0) ? 1.0 : 1.0 / sum;
#pragma unroll
    for (int q = 0; q < TK_MAX_TOP / 64; ++q) if (q * 64 + tid < K) { st[q * 64 + tid] = t[q] * scale; slt[q * 64 + tid] = lt[q] - logsum; }
    if (tid == 0) {
      steacher[0] = !TAIL && sum > 0.0 ? 1.0 : sum;
      steacher[1] = TAIL ? (sum > 1.0 ? 0.0 : 1.0 - sum) : 0.0;
    }
  }
  __syncthreads();
  if constexpr (TAIL) if (tid < 64) {         // the top tokens' own (maximum, sum), each token once
    float m = -INFINITY;
    for (int k = tid; k < K; k += 64) if (sfirst[k]) m = fmaxf(m, sz[k]);
    m = wave_max(m);
    double s = 0.0;
    for (int k = tid; k < K; k += 64) if (sfirst[k]) s += (double)tk_exp2((sz[k] - tk_base(m)) * a.c);
    s = wave_sum(s);
    if (tid == 0) stop = MS{m, s};
  }

  // statistics of the row (TAIL: of what lies outside top)
  float m = xe;
  if constexpr (TAIL) { if (tid < rem) { const int e = nfull * VEC + tid; if (bits[e >> 5] >> (e & 31) & 1) m = -INFINITY; } }
  const float xs = m;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if constexpr (TAIL) {
      const int v = i * T + tid, e = v * VEC;
      const uint32_t top = v < nfull ? bits[e >> 5] >> (e & 31) & ((1u << VEC) - 1) : 0u;
      if (top) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) if (top >> j & 1) {
          if constexpr (ES == 4) x[i].w[j] = TK_NEG<DT>;
          else x[i].w[j >> 1] = j & 1 ? (x[i].w[j >> 1] & 0xffffu) | (TK_NEG<DT> & 0xffff0000u) : (x[i].w[j >> 1] & 0xffff0000u) | (TK_NEG<DT> & 0xffffu);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) m = fmaxf(m, tk_get<DT>(x[i], j));
  }
  float s = tk_exp2((xs - tk_base(m)) * a.c);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    tk_redecode(x[i]);
    float p = 0.0f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) p += tk_exp2((tk_get<DT>(x[i], j) - tk_base(m)) * a.c);
    s += p;
  }
  for (int v = NV * T + tid; v < nfull; v += T) {   // what does not stay: running maximum and sum
    const Pack y = tk_load16(row + (size_t)v * 16);
    uint32_t top = 0;
    if constexpr (TAIL) { const int e = v * VEC; top = bits[e >> 5] >> (e & 31) & ((1u << VEC) - 1); }
    float z[VEC], nm = m;
#pragma unroll
    for (int j = 0; j < VEC; ++j) { z[j] = top >> j & 1 ? -INFINITY : tk_get<DT>(y, j); nm = fmaxf(nm, z[j]); }
    const float b = tk_base(nm);
    float p = 0.0f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) p += tk_exp2((z[j] - b) * a.c);
    s = s * tk_exp2((m - b) * a.c) + p;
    m = nm;
  }
  const MS ms = block_lse<T>(m, s, a.c, red);
  if constexpr (T == 64) __syncthreads();   // (stop; a wider block has passed one in block_lse)
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
  if (S == 0.0 || (!TAIL && sumT == 0.0)) return zeros();   // nothing in the student's row, or nothing in the teacher's (S, sumT: the same for every thread)
  if (tid < 64) {
    const double logS = log(S);
    double l = 0.0;
    for (int k = tid; k < K; k += 64) if (st[k] != 0.0) l += st[k] * (slt[k] - (((double)sz[k] - (double)M) * a.inv_tau - logS));
    l = wave_sum(l);
    if (tid == 0) {
      if (tT > 0.0) l += tT * (log(tT) - (((double)ms.m - (double)M) * a.inv_tau + log(ms.s) - logS));
      a.loss[r] = (float)((double)w * a.tau * a.tau * l);
    }
  }
  if (!grow) return;
  const double wt = (double)w * a.tau;
  float ref, coef;
  if constexpr (TAIL) {
    ref = tk_base(ms.m);   // exp2((z - ref) c) <= 1 for every token outside top
    const double sT = ms.s * (double)tk_exp2((ms.m - tk_base(M)) * a.c) / S;   // their probability
    coef = ms.m == -INFINITY ? 0.0f : (float)(wt * ((sumT + tT) * sT - tT) / ms.s);
  } else {
    ref = tk_base(M);
    coef = (float)(wt * sumT / S);
  }
  // (an infinite exp2 of a top token is overwritten below; a NaN in the row has made coef NaN)
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = i * T + tid;
    if (v < nfull) {
      tk_redecode(x[i]);
      Pack g;
#pragma unroll
      for (int j = 0; j < VEC; j += 2) tk_put2<DT>(g, j, coef * tk_exp2((tk_get<DT>(x[i], j) - ref) * a.c), coef * tk_exp2((tk_get<DT>(x[i], j + 1) - ref) * a.c));
      tk_store16(grow + (size_t)v * 16, g);
    }
  }
  for (int v = NV * T + tid; v < nfull; v += T) {
    const Pack y = tk_load16(row + (size_t)v * 16);
    Pack g;
#pragma unroll
    for (int j = 0; j < VEC; j += 2) tk_put2<DT>(g, j, coef * tk_exp2((tk_get<DT>(y, j) - ref) * a.c), coef * tk_exp2((tk_get<DT>(y, j + 1) - ref) * a.c));
    tk_store16(grow + (size_t)v * 16, g);
  }
  if (tid < rem) tk_set<DT>(grow, nfull * VEC + tid, coef * tk_exp2((xe - ref) * a.c));
  __syncthreads();   // the stream's stores come before the top tokens'
  for (int k = tid; k < K; k += T) {
    if (!sfirst[k]) continue;
    const int t = sidx[k];
    double d = 0.0;
    for (int j = k; j < K; ++j) if (sidx[j] == t) d += st[j];   // a token in several slots: all of their t_k
    const double sk = (double)tk_exp2((sz[k] - tk_base(M)) * a.c) / S;
    tk_set<DT>(grow, t, (float)(wt * (sk * (sumT + tT) - d)));
  }
}

template <int DT, int T, int NV>
void distill_launch(const DistillArgs& a, int rows, hipStream_t st) {
  if (a.lse) hipLaunchKernelGGL((distill_kernel<DT, T, NV, true>), dim3(rows), dim3(T), ((a.V + 31) / 32) * 4, st, a);
  else hipLaunchKernelGGL((distill_kernel<DT, T, NV, false>), dim3(rows), dim3(T), 0, st, a);
}
// the smallest block and register tile that hold the row (a wave holds K slots' threads up to 64); a row beyond 1024 x 16 vectors (256 KB) is held as far as that goes
template <int DT>
void distill_dispatch(const DistillArgs& a, int rows, hipStream_t st) {
  const int nv = (a.V + Lg<DT>::VEC - 1) / Lg<DT>::VEC;
  if (nv <= 64) distill_launch<DT, 64, 1>(a, rows, st);
  else if (nv <= 4 * 256) distill_launch<DT, 256, 4>(a, rows, st);
  else if (nv <= 16 * 256) distill_launch<DT, 256, 16>(a, rows, st);
  else distill_launch<DT, 1024, 16>(a, rows, st);
}

// ------------------------------------------------------------------------------------------ the K largest logits of a row
// Keys: (order of the fp32 value, 19 bits of 2^19 - 1 - index): unique, and their order is "larger value first, equal values by rising index".
// A block streams its row (or its share of one: few rows are split and joined) in chunks of 16 elements a thread, with the running maximum and
// sum a thread for the log-sum-exp, and appends what beats the threshold to a buffer in LDS.  The threshold comes from the chunk itself: the
// K-th largest of the threads' maxima has K elements at or above it, and with T >= 4 K threads few more (1.15 K of random data, at most 16 K
// of any, which is what the buffer has room for).  An element that only equals the threshold comes behind K others and is left out.
// A full buffer is cut by the same rule on its own keys, until each thread holds one and the cut is exact.
struct TopArgs {
  const char* logits; int64_t ld;
  int32_t* idx; float* val; float* lse;
  uint64_t* ws_keys; MS* ws_ms;              // with nsplit > 1: [row][split][K] and [row][split]
  int V, K, nsplit, cap;                     // cap = 16 K + T keys
  float c;
  double inv_tau;
};
__device__ __forceinline__ uint32_t top_order(float v) {   // unsigned order of the values; -0 becomes +0
  const uint32_t u = __float_as_uint(v + 0.0f);
  return u ^ (uint32_t)(((int32_t)u >> 31) | (int32_t)0x80000000);
}
__device__ __forceinline__ float top_value(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }
__device__ __forceinline__ uint64_t top_key(float v, int e) { return ((uint64_t)top_order(v) << 19) | (uint32_t)(TK_MAX_VOCAB - 1 - e); }
constexpr int TOP_KEY_BITS = 51;

// the largest bound that K of the block's T keys (0: none) reach, or 0 where fewer are there.  The first wave's work.
template <int T> __device__ uint64_t top_bound(uint64_t key, int K, uint64_t* sk, uint64_t* sbound) {
  sk[threadIdx.x] = key;
  __syncthreads();
  if (threadIdx.x < 64) {
    uint64_t k[T / 64];
#pragma unroll
    for (int i = 0; i < T / 64; ++i) k[i] = sk[i * 64 + threadIdx.x];
    uint64_t b = 0;
    for (int bit = TOP_KEY_BITS - 1; bit >= 0; --bit) {
      const uint64_t cand = b | (1ull << bit);
      int n = 0;
#pragma unroll
      for (int i = 0; i < T / 64; ++i) n += __popcll(__ballot(k[i] >= cand));
      if (n >= K) b = cand;
      if (n == K) break;
    }
    if (threadIdx.x == 0) *sbound = b;
  }
  __syncthreads();
  const uint64_t b = *sbound;
  __syncthreads();
  return b;
}
// the buffer's n <= 5 T keys cut to at most T, the K largest among them; returns their number and raises the bar
template <int T> __device__ int top_cut(uint64_t* buf, int n, int K, float* bar, int* sfill, uint64_t* sk, uint64_t* sbound) {
  constexpr int MOST = 5;   // cap = 16 K + T keys, K <= T / 4
  while (n > T) {
    uint64_t k[MOST], best = 0;
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
      k[i] = i * T + (int)threadIdx.x < n ? buf[i * T + threadIdx.x] : 0;
      best = k[i] > best ? k[i] : best;
    }
    const uint64_t bound = top_bound<T>(best, K, sk, sbound);   // (its barriers stand between the reads above and the writes below)
    if (bound) *bar = fmaxf(*bar, top_value((uint32_t)(bound >> 19)));
    if (threadIdx.x == 0) *sfill = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MOST; ++i) if (k[i] != 0 && k[i] >= bound) buf[atomicAdd(sfill, 1)] = k[i];
    __syncthreads();
    n = *sfill;
    __syncthreads();
  }
  return n;
}
// writes the buffer's K largest in order; n <= T
template <int T> __device__ void top_write(const uint64_t* buf, int n, int K, int32_t* idx, float* val, uint64_t* keys) {
  if ((int)threadIdx.x < n) {
    const uint64_t mine = buf[threadIdx.x];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += buf[j] > mine;
    if (rank < K) {
      if (keys) keys[rank] = mine;
      else { idx[rank] = TK_MAX_VOCAB - 1 - (int)(mine & (TK_MAX_VOCAB - 1)); val[rank] = top_value((uint32_t)(mine >> 19)); }
    }
  }
  for (int k = n + (int)threadIdx.x; k < K; k += T) {
    if (keys) keys[k] = 0;
    else { idx[k] = -1; val[k] = -INFINITY; }
  }
}
__device__ __forceinline__ float top_lse(MS ms, double inv_tau) {
  if (ms.m == -INFINITY && ms.s == 0.0) return -INFINITY;
  if (ms.m == INFINITY) return INFINITY;
  return (float)((double)tk_base(ms.m) * inv_tau + log(ms.s));
}

template <int DT, int T>
__global__ __launch_bounds__(T) void top_kernel(TopArgs a) {
  constexpr int VEC = Lg<DT>::VEC, U = 16 / VEC;
  extern __shared__ uint64_t buf[];          // [cap]
  __shared__ uint64_t sk[T];
  __shared__ uint64_t sbound;
  __shared__ MS red[T / 64];
  __shared__ int scount[3], sfill;
  const int tid = threadIdx.x, V = a.V, K = a.K;
  const int64_t r = blockIdx.x / (uint32_t)a.nsplit;
  const int split = (int)(blockIdx.x - r * a.nsplit);
  const char* row = a.logits + r * a.ld;
  const int nvec = (V + VEC - 1) / VEC, nchunk = (nvec + T * U - 1) / (T * U);
  const int c0 = (int)((int64_t)nchunk * split / a.nsplit), c1 = (int)((int64_t)nchunk * (split + 1) / a.nsplit);
  if (tid < 3) scount[tid] = 0;
  if (tid == 3) sfill = 0;
  __syncthreads();
  float bar = -INFINITY;                     // an element has to be above it
  int fill = 0;                              // keys in the buffer
  float m = -INFINITY, s = 0.0f;
  Pack x[U], y[U];
#pragma unroll
  for (int u = 0; u < U; ++u) y[u] = c0 < c1 ? tk_load<DT>(row, (c0 * U + u) * T + tid, V) : tk_neg<DT>();
  int turn = 0;                              // which of the three counters
  for (int ch = c0; ch < c1; ++ch) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      x[u] = y[u];
      if (ch + 1 < c1) y[u] = tk_load<DT>(row, ((ch + 1) * U + u) * T + tid, V);
    }
    float cm = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) cm = fmaxf(cm, tk_get<DT>(x[u], j));
    const float nm = fmaxf(m, cm), b = tk_base(nm);
    float p = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) p += tk_exp2((tk_get<DT>(x[u], j) - b) * a.c);
    s = s * tk_exp2((m - b) * a.c) + p;
    m = nm;
    // how many of the chunk's elements are above the bar
    const auto above = [&] {
      int n = 0;
      if (cm > bar) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < VEC; ++j) n += tk_get<DT>(x[u], j) > bar;
        atomicAdd(&scount[turn], n);
      }
      __syncthreads();
      const int t = scount[turn];
      if (tid == 0) scount[turn == 0 ? 2 : turn - 1] = 0;   // the counter of the turn before: nobody reads it any more, and two barriers pass until it counts again
      turn = turn == 2 ? 0 : turn + 1;
      return t;
    };
    int n = above();
    if (n == 0) continue;
    uint64_t bound = 0;
    if (fill + n > a.cap) {
      if (fill > T) {
        fill = top_cut<T>(buf, fill, K, &bar, &sfill, sk, &sbound);
        n = above();
      }
      if (fill + n > a.cap) {
        uint64_t best = 0;
        if (cm > bar) {
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = VEC - 1; j >= 0; --j) {
              const float z = tk_get<DT>(x[u], j);
              if (z == cm) { const uint64_t k = top_key(z, ((ch * U + u) * T + tid) * VEC + j); best = k > best ? k : best; }
            }
        }
        bound = top_bound<T>(best, K, sk, &sbound);
      }
    }
    if (cm > bar) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float z = tk_get<DT>(x[u], j);
          if (z > bar) {
            const uint64_t k = top_key(z, ((ch * U + u) * T + tid) * VEC + j);
            if (k >= bound) { const int at = atomicAdd(&sfill, 1); if (at < a.cap) buf[at] = k; }
          }
        }
    }
    if (bound) bar = fmaxf(bar, top_value((uint32_t)(bound >> 19)));
    __syncthreads();
    fill = sfill;
  }
  __syncthreads();
  fill = top_cut<T>(buf, fill, K, &bar, &sfill, sk, &sbound);
  const MS ms = block_lse<T>(m, s, a.c, red);
  if (a.nsplit > 1) {
    top_write<T>(buf, fill, K, nullptr, nullptr, a.ws_keys + (r * a.nsplit + split) * K);
    if (tid == 0) a.ws_ms[r * a.nsplit + split] = ms;
  } else {
    top_write<T>(buf, fill, K, a.idx + r * K, a.val + r * K, nullptr);
    if (tid == 0) a.lse[r] = top_lse(ms, a.inv_tau);
  }
}
// the splits of a row: their keys are one more buffer to cut
template <int T>
__global__ __launch_bounds__(T) void top_join_kernel(TopArgs a) {
  extern __shared__ uint64_t buf[];
  __shared__ uint64_t sk[T];
  __shared__ uint64_t sbound;
  __shared__ int sfill;
  const int tid = threadIdx.x, K = a.K;
  const int64_t r = blockIdx.x;
  if (tid == 0) sfill = 0;
  __syncthreads();
  for (int i = tid; i < a.nsplit * K; i += T) {
    const uint64_t k = a.ws_keys[r * a.nsplit * K + i];
    if (k) buf[atomicAdd(&sfill, 1)] = k;
  }
  __syncthreads();
  int fill = sfill;
  float bar = -INFINITY;
  __syncthreads();
  fill = top_cut<T>(buf, fill, K, &bar, &sfill, sk, &sbound);
  top_write<T>(buf, fill, K, a.idx + r * K, a.val + r * K, nullptr);
  if (tid == 0) {
    MS ms = a.ws_ms[r * a.nsplit];
    for (int i = 1; i < a.nsplit; ++i) {
      const MS o = a.ws_ms[r * a.nsplit + i];
      const float M = fmaxf(ms.m, o.m), B = tk_base(M);
      ms.s = ms.s * (double)tk_exp2((ms.m - B) * a.c) + o.s * (double)tk_exp2((o.m - B) * a.c);
      ms.m = M;
    }
    a.lse[r] = top_lse(ms, a.inv_tau);
  }
}
struct TopPlan { int threads, nsplit, cap; size_t lds, ws; };
TopPlan top_plan(int rows, int V, int K, int es) {
  TopPlan p;
  p.threads = K <= 16 && V <= 1024 ? 64 : (K <= 64 ? 256 : (K <= 128 ? 512 : 1024));   // T >= 4 K
  p.cap = 16 * K + p.threads;
  const int chunk = p.threads * 16, nchunk = (V + chunk - 1) / chunk;
  // few rows: split until there are about 512 blocks; the join holds nsplit K <= cap keys
  int n = rows >= 512 ? 1 : (512 + rows - 1) / rows;
  n = n < nchunk ? n : nchunk;
  n = n < p.cap / K ? n : p.cap / K;
  p.nsplit = n < 16 ? n : 16;
  p.lds = (size_t)p.cap * 8;
  p.ws = p.nsplit > 1 ? (size_t)rows * p.nsplit * ((size_t)K * 8 + sizeof(MS)) : 0;
  (void)es;
  return p;
}
template <int DT, int T> void top_launch(const TopArgs& a, int rows, const TopPlan& p, hipStream_t st) {
  hipLaunchKernelGGL((top_kernel<DT, T>), dim3((uint32_t)rows * p.nsplit), dim3(T), p.lds, st, a);
  if (p.nsplit > 1) hipLaunchKernelGGL(top_join_kernel<T>, dim3(rows), dim3(T), p.lds, st, a);
}
template <int DT> void top_dispatch(const TopArgs& a, int rows, const TopPlan& p, hipStream_t st) {
  if (p.threads == 64) top_launch<DT, 64>(a, rows, p, st);
  else if (p.threads == 256) top_launch<DT, 256>(a, rows, p, st);
  else if (p.threads == 512) top_launch<DT, 512>(a, rows, p, st);
  else top_launch<DT, 1024>(a, rows, p, st);
}

// ------------------------------------------------------------------------------------------ drafted tokens against the target
// p_i = softmax(target row i / tau), q_i = softmax(draft row i / tau), or one-hot at the drafted token where there are no draft logits.
//   accepted while u_i q_i(x_i) < p_i(x_i), i < n;  at the first rejection a the next token is drawn from max(p_a - q_a, 0) (from p_a where that has
//   no mass), after n acceptances from p_n: the first token whose cumulative weight exceeds u_s times the whole.
// An acceptance compares two numbers; a drawn token lies between two neighbours of a cumulative sum over the whole vocabulary, so that the row the token
// is drawn from is summed in fp64 throughout (exps too), chunk by chunk of 4096 tokens, and the statistics of all other rows with fp32 exps.
//   verify_stats_kernel   (maximum, sum) of the rows of every drafted position, split over blocks
//   verify_sums_kernel    acceptance (each block of a sequence for itself), then the chunks' fp64 sums of the row that the token is drawn from
//   verify_rest_kernel    the chunks' sums of max(p - q, 0), where the sequence has a rejection and a draft distribution
//   verify_pick_kernel    the chunk, then the token inside it
constexpr int VF_T = 256, VF_CHUNK = 4096;   // 16 tokens a thread
struct VerifyArgs {
  const char* target; int64_t tb, tp;        // bytes from sequence to sequence, from position to position
  const char* draft; int64_t db, dp;         // null: no draft distribution
  const int32_t* tokens; const int32_t* n_draft; const float* u_accept; const float* u_sample;
  int32_t* out; int32_t* accepted; float* logprobs;
  MS* stats;                                 // [position][sequence][target, draft][split]
  struct VfSum* sums;                        // [sequence][chunk]
  double* rest;                              // [sequence][chunk]
  int B, K, V, nsplit, nchunk;
  float c;
  double inv_tau;
};
struct VfSum { double p, q; float mp, mq; }; // sums of exp((z - m) / tau) over a chunk, and its maxima; without draft logits q is what the rejected token alone adds to p
__device__ __forceinline__ int vf_drafts(const VerifyArgs& a, int b) {
  const int n = a.n_draft ? a.n_draft[b] : a.K;
  return n < 0 ? 0 : (n > a.K ? a.K : n);
}

template <int DT>
__global__ __launch_bounds__(VF_T) void verify_stats_kernel(VerifyArgs a) {
  constexpr int VEC = Lg<DT>::VEC, U = 4;
  __shared__ MS red[VF_T / 64];
  const int rows = a.draft ? 2 : 1;
  uint32_t id = blockIdx.x;
  const int split = (int)(id % (uint32_t)a.nsplit); id /= (uint32_t)a.nsplit;
  const int which = (int)(id % (uint32_t)rows); id /= (uint32_t)rows;
  const int b = (int)(id % (uint32_t)a.B), i = (int)(id / (uint32_t)a.B);
  if (i >= vf_drafts(a, b)) return;
  const char* row = which ? a.draft + b * a.db + i * a.dp : a.target + b * a.tb + i * a.tp;
  const int nvec = (a.V + VEC - 1) / VEC;
  const int v0 = (int)((int64_t)nvec * split / a.nsplit), v1 = (int)((int64_t)nvec * (split + 1) / a.nsplit);
  float m = -INFINITY, s = 0.0f;
  for (int v = v0; v < v1; v += VF_T * U) {
    Pack x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) { const int at = v + u * VF_T + (int)threadIdx.x; x[u] = at < v1 ? tk_load<DT>(row, at, a.V) : tk_neg<DT>(); }
    float nm = m;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) nm = fmaxf(nm, tk_get<DT>(x[u], j));
    const float base = tk_base(nm);
    float p = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) p += tk_exp2((tk_get<DT>(x[u], j) - base) * a.c);
    s = s * tk_exp2((m - base) * a.c) + p;
    m = nm;
  }
  const MS ms = block_lse<VF_T>(m, s, a.c, red);
  if (threadIdx.x == 0) a.stats[blockIdx.x] = ms;
}

// probability of `token` in a row whose statistics are split; NaN where the row is no distribution (nothing but -inf, a NaN, +inf)
template <int DT> __device__ double vf_prob(const VerifyArgs& a, const MS* st, const char* row, int token, double* logp) {
  float M = st[0].m;
  for (int k = 1; k < a.nsplit; ++k) M = fmaxf(M, st[k].m);
  double S = 0.0;
  for (int k = 0; k < a.nsplit; ++k) S += st[k].s * (double)tk_exp2((st[k].m - tk_base(M)) * a.c);
  if (!(M > -INFINITY && M < INFINITY)) return NAN;
  const double x = ((double)tk_at<DT>(row, token) - (double)M) * a.inv_tau;
  *logp = x - log(S);
  return exp(x) / S;
}

template <int DT>
__global__ __launch_bounds__(VF_T) void verify_sums_kernel(VerifyArgs a) {
  constexpr int VEC = Lg<DT>::VEC, U = 16 / VEC;
  __shared__ int sa;
  __shared__ float sm[2][VF_T / 64];
  __shared__ double ss[2][VF_T / 64];
  const int tid = threadIdx.x;
  const int b = (int)(blockIdx.x / (uint32_t)a.nchunk), ch = (int)(blockIdx.x % (uint32_t)a.nchunk);
  const int n = vf_drafts(a, b);
  if (tid == 0) sa = n;
  __syncthreads();
  double logp = 0.0;
  int x = -1;
  if (tid < n) {
    x = a.tokens[(int64_t)b * a.K + tid];
    bool ok = false;
    if ((uint32_t)x < (uint32_t)a.V) {
      const int rows = a.draft ? 2 : 1;
      const MS* st = a.stats + ((int64_t)(tid * a.B + b) * rows) * a.nsplit;
      const double p = vf_prob<DT>(a, st, a.target + b * a.tb + tid * a.tp, x, &logp);
      double q = 1.0, unused;
      if (a.draft) q = vf_prob<DT>(a, st + a.nsplit, a.draft + b * a.db + tid * a.dp, x, &unused);
      ok = (double)a.u_accept[(int64_t)b * a.K + tid] * q < p;   // (a NaN on either side: not accepted)
    }
    if (!ok) atomicMin(&sa, tid);
  }
  __syncthreads();
  const int at = sa;
  if (ch == 0) {
    if (tid < at) { a.out[(int64_t)b * (a.K + 1) + tid] = x; if (a.logprobs) a.logprobs[(int64_t)b * (a.K + 1) + tid] = (float)logp; }
    else if (tid > at && tid <= a.K) { a.out[(int64_t)b * (a.K + 1) + tid] = -1; if (a.logprobs) a.logprobs[(int64_t)b * (a.K + 1) + tid] = 0.0f; }
    if (tid == 0) a.accepted[b] = at;
  }
  // the row that the next token is drawn from, and the draft's row where a token was rejected
  const char* prow = a.target + b * a.tb + at * a.tp;
  const char* qrow = a.draft && at < n ? a.draft + b * a.db + at * a.dp : nullptr;
  const int skip = !a.draft && at < n ? a.tokens[(int64_t)b * a.K + at] : -1;   // a looked-up token that was rejected has no weight left
  Pack px[U], qx[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int v = (ch * U + u) * VF_T + tid;
    px[u] = tk_load<DT>(prow, v, a.V);
    qx[u] = qrow ? tk_load<DT>(qrow, v, a.V) : tk_neg<DT>();
  }
  float mp = -INFINITY, mq = -INFINITY;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < VEC; ++j) { mp = fmaxf(mp, tk_get<DT>(px[u], j)); mq = fmaxf(mq, tk_get<DT>(qx[u], j)); }
  mp = wave_max(mp); mq = wave_max(mq);
  if ((tid & 63) == 0) { sm[0][tid >> 6] = mp; sm[1][tid >> 6] = mq; }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < VF_T / 64; ++i) { mp = fmaxf(mp, sm[0][i]); mq = fmaxf(mq, sm[1][i]); }
  double sp = 0.0, sq = 0.0;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const double e = exp(((double)tk_get<DT>(px[u], j) - (double)tk_base(mp)) * a.inv_tau);
      if (((ch * U + u) * VF_T + tid) * VEC + j == skip) sq = e; else sp += e;
      if (qrow) sq += exp(((double)tk_get<DT>(qx[u], j) - (double)tk_base(mq)) * a.inv_tau);
    }
  sp = wave_sum(sp); sq = wave_sum(sq);
  if ((tid & 63) == 0) { ss[0][tid >> 6] = sp; ss[1][tid >> 6] = sq; }
  __syncthreads();
  if (tid == 0) {
    sp = sq = 0.0;
    for (int i = 0; i < VF_T / 64; ++i) { sp += ss[0][i]; sq += ss[1][i]; }
    a.sums[blockIdx.x] = VfSum{sp, sq, mp, mq};
  }
}

// a sequence's row as a whole: maximum, sum, and whether it is a distribution
struct VfRow { double m, s; bool good; };
__device__ __forceinline__ VfRow vf_row(const VerifyArgs& a, int b, bool q) {
  const VfSum* s = a.sums + (int64_t)b * a.nchunk;
  float M = -INFINITY;
  for (int i = 0; i < a.nchunk; ++i) M = fmaxf(M, q ? s[i].mq : s[i].mp);
  double S = 0.0;
  for (int i = 0; i < a.nchunk; ++i) S += (q ? s[i].q : (a.draft ? s[i].p : s[i].p + s[i].q)) * exp(((double)(q ? s[i].mq : s[i].mp) - (double)tk_base(M)) * a.inv_tau);
  return VfRow{(double)M, S, M > -INFINITY && M < INFINITY && S > 0.0};
}
// the weight of a token: p, max(p - q, 0), or p without the rejected token of a looked-up draft
struct VfWeight {
  double inv_tau, pm, pn, qm, qn;            // pn, qn: 1 / sum
  int skip;                                  // a token of no weight, or -1
  bool q;
  __device__ double operator()(float zp, float zq, int e) const {
    const double p = exp(((double)zp - pm) * inv_tau) * pn;
    if (q) { const double d = p - exp(((double)zq - qm) * inv_tau) * qn; return d > 0.0 ? d : 0.0; }
    return e == skip ? 0.0 : p;
  }
};

template <int DT>
__global__ __launch_bounds__(VF_T) void verify_rest_kernel(VerifyArgs a) {
  constexpr int VEC = Lg<DT>::VEC, U = 16 / VEC;
  __shared__ double ss[VF_T / 64];
  __shared__ VfRow srow[2];
  const int tid = threadIdx.x;
  const int b = (int)(blockIdx.x / (uint32_t)a.nchunk), ch = (int)(blockIdx.x % (uint32_t)a.nchunk);
  const int at = a.accepted[b];
  if (at >= vf_drafts(a, b)) return;
  if (tid < 2) srow[tid] = vf_row(a, b, tid == 1);
  __syncthreads();
  if (!srow[0].good || !srow[1].good) return;
  const VfWeight w = {a.inv_tau, srow[0].m, 1.0 / srow[0].s, srow[1].m, 1.0 / srow[1].s, -1, true};
  const char* prow = a.target + b * a.tb + at * a.tp;
  const char* qrow = a.draft + b * a.db + at * a.dp;
  double s = 0.0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int v = (ch * U + u) * VF_T + tid;
    const Pack px = tk_load<DT>(prow, v, a.V), qx = tk_load<DT>(qrow, v, a.V);
#pragma unroll
    for (int j = 0; j < VEC; ++j) s += w(tk_get<DT>(px, j), tk_get<DT>(qx, j), 0);
  }
  s = wave_sum(s);
  if ((tid & 63) == 0) ss[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) { s = 0.0; for (int i = 0; i < VF_T / 64; ++i) s += ss[i]; a.rest[blockIdx.x] = s; }
}

template <int DT>
__global__ __launch_bounds__(VF_T) void verify_pick_kernel(VerifyArgs a) {
  constexpr int PER = VF_CHUNK / VF_T;       // neighbouring tokens a thread
  __shared__ VfRow srow[2];
  __shared__ VfWeight sweight;
  __shared__ double sbelow, sgoal, ss[VF_T / 64];
  __shared__ int schunk, stoken, slast;
  const int tid = threadIdx.x, b = blockIdx.x;
  const int n = vf_drafts(a, b), at = a.accepted[b];
  const int64_t o = (int64_t)b * (a.K + 1) + at;
  const char* prow = a.target + b * a.tb + at * a.tp;
  const char* qrow = a.draft && at < n ? a.draft + b * a.db + at * a.dp : nullptr;
  const VfSum* sums = a.sums + (int64_t)b * a.nchunk;
  if (tid == 0 || (tid == 1 && qrow)) srow[tid] = vf_row(a, b, tid == 1);
  if (tid == 0) { stoken = a.V; slast = -1; }
  __syncthreads();
  if (!srow[0].good) {                       // no distribution to draw from
    if (tid == 0) { a.out[o] = -1; if (a.logprobs) a.logprobs[o] = 0.0f; }
    return;
  }
  if (tid == 0) {
    VfWeight w = {a.inv_tau, srow[0].m, 1.0 / srow[0].s, 0.0, 0.0, -1, false};
    const int x = at < n ? a.tokens[(int64_t)b * a.K + at] : -1;
    if (qrow && srow[1].good) {
      w.q = true; w.qm = srow[1].m; w.qn = 1.0 / srow[1].s;
      double total = 0.0;
      for (int i = 0; i < a.nchunk; ++i) total += a.rest[(int64_t)b * a.nchunk + i];
      if (!(total > 0.0)) w.q = false;       // p nowhere above q
    } else if (!a.draft && (uint32_t)x < (uint32_t)a.V) w.skip = x;
    double total = 0.0;
    const auto chunk = [&](int i) {
      if (w.q) return a.rest[(int64_t)b * a.nchunk + i];
      return (!a.draft && w.skip < 0 ? sums[i].p + sums[i].q : sums[i].p) * exp(((double)sums[i].mp - w.pm) * a.inv_tau) * w.pn;
    };
    for (int i = 0; i < a.nchunk; ++i) total += chunk(i);
    if (!(total > 0.0)) { w.skip = -1; total = 0.0; for (int i = 0; i < a.nchunk; ++i) total += chunk(i); }
    const float u = a.u_sample[b];
    const double goal = (u > 0.0f ? (double)u : 0.0) * total;
    double below = 0.0, start = 0.0;
    int hit = -1;
    for (int i = 0; i < a.nchunk; ++i) {     // the first chunk that ends above the goal; the last one with weight where rounding (or u >= 1) leaves none
      const double s = chunk(i);
      if (s > 0.0) {
        hit = i; start = below;
        if (below + s > goal) break;
      }
      below += s;
    }
    schunk = hit; sbelow = start; sgoal = goal; sweight = w;
  }
  __syncthreads();
  const VfWeight w = sweight;
  const int e0 = schunk * VF_CHUNK + tid * PER;
  double t[PER], s = 0.0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = e0 + j;
    t[j] = e < a.V ? w(tk_at<DT>(prow, e), w.q ? tk_at<DT>(qrow, e) : 0.0f, e) : 0.0;
    s += t[j];
  }
  // exclusive sum over the threads before
  double inc = s;
  for (int d = 1; d < 64; d <<= 1) { const double v = __shfl_up(inc, d, 64); if ((tid & 63) >= d) inc += v; }
  if ((tid & 63) == 63) ss[tid >> 6] = inc;
  __syncthreads();
  double c = sbelow + (inc - s);
  for (int i = 0; i < (tid >> 6); ++i) c += ss[i];
  int first = a.V, last = -1;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    c += t[j];
    if (t[j] > 0.0) { last = e0 + j; if (c > sgoal && first == a.V) first = e0 + j; }
  }
  if (first < a.V) atomicMin(&stoken, first);
  if (last >= 0) atomicMax(&slast, last);
  __syncthreads();
  if (tid == 0) {
    const int token = stoken < a.V ? stoken : slast;
    a.out[o] = token;
    if (a.logprobs) a.logprobs[o] = token < 0 ? 0.0f : (float)(((double)tk_at<DT>(prow, token) - srow[0].m) * a.inv_tau - log(srow[0].s));
  }
}

// tau = 0: p is one-hot at the row's largest logit (the lowest index of equal ones), a draft is accepted where it is that token
struct VfBest { float m; int32_t idx, bad, pad; };   // bad: a NaN or +inf among the logits
static_assert(sizeof(VfBest) == sizeof(MS), "both live in the same part of the workspace");
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
    reinterpret_cast<VfBest*>(a.stats)[blockIdx.x] = VfBest{m, idx, bad, 0};
  }
}
__global__ __launch_bounds__(VF_T) void verify_greedy_kernel(VerifyArgs a) {
  __shared__ int sa;
  const int tid = threadIdx.x, b = blockIdx.x, n = vf_drafts(a, b);
  if (tid == 0) sa = n;
  __syncthreads();
  int best = -1;
  if (tid <= n) {
    const VfBest* st = reinterpret_cast<const VfBest*>(a.stats) + ((int64_t)tid * a.B + b) * a.nsplit;
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

struct VerifyPlan { int nsplit, nchunk; size_t o_sums, o_rest, ws; };
VerifyPlan verify_plan(int B, int K, int V, int es, bool draft, bool greedy) {
  VerifyPlan p;
  const int nvec = (int)(((int64_t)V * es + 15) / 16);
  const int64_t rows = greedy ? (int64_t)B * (K + 1) : (int64_t)B * K * (draft ? 2 : 1);
  // about 1024 blocks in all, a share of at least 1024 vectors each
  int64_t n = rows > 0 ? (1024 + rows - 1) / rows : 1;
  const int most = (nvec + 1023) / 1024;
  p.nsplit = (int)(n < most ? n : most);
  p.nchunk = (V + VF_CHUNK - 1) / VF_CHUNK;
  p.o_sums = (size_t)rows * p.nsplit * sizeof(MS);
  p.o_rest = p.o_sums + (greedy ? 0 : (size_t)B * p.nchunk * sizeof(VfSum));
  p.ws = p.o_rest + (greedy ? 0 : (size_t)B * p.nchunk * sizeof(double));
  return p;
}
template <int DT> void verify_dispatch(const VerifyArgs& a, bool greedy, hipStream_t st) {
  if (greedy) {
    hipLaunchKernelGGL(verify_best_kernel<DT>, dim3((uint32_t)((int64_t)a.B * (a.K + 1) * a.nsplit)), dim3(VF_T), 0, st, a);
    hipLaunchKernelGGL(verify_greedy_kernel, dim3(a.B), dim3(VF_T), 0, st, a);
    return;
  }
  const uint32_t rows = (uint32_t)((int64_t)a.B * a.K * (a.draft ? 2 : 1));
  if (rows) hipLaunchKernelGGL(verify_stats_kernel<DT>, dim3(rows * (uint32_t)a.nsplit), dim3(VF_T), 0, st, a);
  hipLaunchKernelGGL(verify_sums_kernel<DT>, dim3((uint32_t)a.B * a.nchunk), dim3(VF_T), 0, st, a);
  if (a.draft && a.K > 0) hipLaunchKernelGGL(verify_rest_kernel<DT>, dim3((uint32_t)a.B * a.nchunk), dim3(VF_T), 0, st, a);
  hipLaunchKernelGGL(verify_pick_kernel<DT>, dim3(a.B), dim3(VF_T), 0, st, a);
}

// ------------------------------------------------------------------------------------------ entry points: checks, plan, launches
#define TK_REFUSE(...) do { cbm_set_error(__VA_ARGS__); return -1; } while (0)
bool tk_temperature(float t) { return t >= 1e-4f && t <= 1e4f; }
int tk_es(int dtype) { return dtype == CBM_F32 ? 4 : 2; }
int tk_rows(const char* fn, int dtype, int64_t rows, int vocab) {
  if (dtype != CBM_F32 && dtype != CBM_BF16 && dtype != CBM_F16) TK_REFUSE("%s: dtype %d is none of CBM_F32, CBM_BF16, CBM_F16", fn, dtype);
  if (vocab < 1 || vocab > TK_MAX_VOCAB) TK_REFUSE("%s: vocab %d outside [1, %d]", fn, vocab, TK_MAX_VOCAB);
  if (rows < 0 || rows > (1 << 24)) TK_REFUSE("%s: %lld rows outside [0, 2^24]", fn, (long long)rows);
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
  return rows ? (int64_t)top_plan(rows, vocab, k, tk_es(dtype)).ws : 0;
}
extern "C" int cbm_top_logits(cbm_ctx* c, const void* logits, int32_t dtype, int32_t rows, int32_t vocab, int64_t row_stride, int32_t k,
                              float temperature, int32_t* idx, float* values, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* fn = "cbm_top_logits";
  if (tk_rows(fn, dtype, rows, vocab)) return -1;
  if (k < 1 || k > TK_MAX_TOP) TK_REFUSE("%s: k %d outside [1, %d]", fn, k, TK_MAX_TOP);
  if (!tk_temperature(temperature)) TK_REFUSE("%s: temperature %g outside [1e-4, 1e4]", fn, temperature);
  if (rows > 1 && row_stride < vocab) TK_REFUSE("%s: row stride %lld is smaller than the vocabulary %d", fn, (long long)row_stride, vocab);
  if (rows == 0) { if (!c) TK_REFUSE("%s: null context", fn); return 0; }
  const int es = tk_es(dtype);
  if (tk_pointer(fn, "logits", logits, es) || tk_pointer(fn, "idx", idx, 4) || tk_pointer(fn, "values", values, 4) || tk_pointer(fn, "lse", lse, 4)) return -1;
  const TopPlan p = top_plan(rows, vocab, k, es);
  if (tk_workspace(fn, workspace, workspace_bytes, p.ws)) return -1;
  if (!c) TK_REFUSE("%s: null context", fn);
  DeviceScope dev(c);
  if (!dev.ok) TK_REFUSE("%s: cannot select device %d", fn, c->cfg.device);
  TopArgs a = {};
  a.logits = (const char*)logits; a.ld = row_stride * es;
  a.idx = idx; a.val = values; a.lse = lse;
  a.ws_keys = (uint64_t*)workspace; a.ws_ms = (MS*)((char*)workspace + (size_t)rows * p.nsplit * k * 8);
  a.V = vocab; a.K = k; a.nsplit = p.nsplit; a.cap = p.cap;
  a.inv_tau = 1.0 / (double)temperature; a.c = (float)(TK_LOG2E * a.inv_tau);
  hipStream_t st = tk_stream(c, stream);
  if (dtype == CBM_F32) top_dispatch<CBM_F32>(a, rows, p, st);
  else if (dtype == CBM_BF16) top_dispatch<CBM_BF16>(a, rows, p, st);
  else top_dispatch<CBM_F16>(a, rows, p, st);
  return tk_done(fn);
}

extern "C" int cbm_distill_loss_grad(cbm_ctx* c, const void* logits, int32_t dtype, int32_t rows, int32_t vocab, int64_t row_stride,
                                     const int32_t* teacher_idx, const float* teacher_logits, int32_t k, const float* teacher_lse,
                                     const float* row_weight, float temperature, float* loss, void* dlogits, int64_t grad_stride, void* stream) {
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
  a.V = vocab; a.K = k;
  a.tau = (double)temperature; a.inv_tau = 1.0 / a.tau; a.c = (float)(TK_LOG2E * a.inv_tau);
  hipStream_t st = tk_stream(c, stream);
  if (dtype == CBM_F32) distill_dispatch<CBM_F32>(a, rows, st);
  else if (dtype == CBM_BF16) distill_dispatch<CBM_BF16>(a, rows, st);
  else distill_dispatch<CBM_F16>(a, rows, st);
  return tk_done(fn);
}

static int verify_check(const char* fn, int dtype, int B, int K, int V, float temperature) {
  if (tk_rows(fn, dtype, B, V)) return -1;
  if (K < 0 || K > TK_MAX_DRAFTS) TK_REFUSE("%s: %d drafts outside [0, %d]", fn, K, TK_MAX_DRAFTS);
  if (!(temperature == 0.0f || tk_temperature(temperature))) TK_REFUSE("%s: temperature %g is neither 0 nor in [1e-4, 1e4]", fn, temperature);
  if ((int64_t)B * (2 * K + 1) > (1 << 24)) TK_REFUSE("%s: %d sequences of %d drafts are more than 2^24 rows", fn, B, K);
  return 0;
}
extern "C" int64_t cbm_verify_drafts_workspace(int32_t dtype, int32_t batch, int32_t drafts, int32_t vocab, int32_t with_draft_logits, float temperature) {
  if (verify_check("cbm_verify_drafts_workspace", dtype, batch, drafts, vocab, temperature)) return -1;
  return batch ? (int64_t)verify_plan(batch, drafts, vocab, tk_es(dtype), with_draft_logits != 0, temperature == 0.0f).ws : 0;
}
extern "C" int cbm_verify_drafts(cbm_ctx* c, const void* target_logits, int32_t dtype, int32_t batch, int32_t drafts, int32_t vocab,
                                 int64_t target_batch_stride, int64_t target_pos_stride, const void* draft_logits, int64_t draft_batch_stride,
                                 int64_t draft_pos_stride, const int32_t* draft_tokens, const int32_t* n_draft, const float* u_accept,
                                 const float* u_sample, float temperature, int32_t* tokens, int32_t* accepted, float* logprobs, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  const char* fn = "cbm_verify_drafts";
  if (verify_check(fn, dtype, batch, drafts, vocab, temperature)) return -1;
  const bool greedy = temperature == 0.0f;
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
  const VerifyPlan p = verify_plan(batch, drafts, vocab, es, draft_logits != nullptr, greedy);
  if (tk_workspace(fn, workspace, workspace_bytes, p.ws)) return -1;
  if (!c) TK_REFUSE("%s: null context", fn);
  DeviceScope dev(c);
  if (!dev.ok) TK_REFUSE("%s: cannot select device %d", fn, c->cfg.device);
  VerifyArgs a = {};
  a.target = (const char*)target_logits; a.tb = target_batch_stride * es; a.tp = target_pos_stride * es;
  a.draft = (const char*)draft_logits; a.db = draft_batch_stride * es; a.dp = draft_pos_stride * es;
  a.tokens = draft_tokens; a.n_draft = n_draft; a.u_accept = u_accept; a.u_sample = u_sample;
  a.out = tokens; a.accepted = accepted; a.logprobs = logprobs;
  a.stats = (MS*)workspace; a.sums = (VfSum*)((char*)workspace + p.o_sums); a.rest = (double*)((char*)workspace + p.o_rest);
  a.B = batch; a.K = drafts; a.V = vocab; a.nsplit = p.nsplit; a.nchunk = p.nchunk;
  a.inv_tau = greedy ? 1.0 : 1.0 / (double)temperature; a.c = (float)(TK_LOG2E * a.inv_tau);
  hipStream_t st = tk_stream(c, stream);
  if (dtype == CBM_F32) verify_dispatch<CBM_F32>(a, greedy, st);
  else if (dtype == CBM_BF16) verify_dispatch<CBM_BF16>(a, greedy, st);
  else verify_dispatch<CBM_F16>(a, greedy, st);
  return tk_done(fn);
}

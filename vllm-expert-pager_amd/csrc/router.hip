// The router beside the experts: the choice of each token's experts from its
// logits, the balance loss with the per-expert counts, and the gradient
// through both.
//
// Choice: a logit that is NaN or -inf is masked. The key of expert i is its
// logit, or, with a selection bias, its score plus the bias. Softmax and the
// sigmoid grow with the logit, so without a bias the order of the logits is
// the order of the scores, free of rounding; with a bias the keys are formed
// in 64 bits, since two 32-bit keys next to each other may round to the wrong
// order. The topk largest keys are taken in descending order, equal keys by
// the lower index; where fewer are left the id is -1 and the weight 0. With
// groups, the best `keep` groups stay, by their largest key, or with a bias
// by the sum of their two largest keys.
//
// Weights: score_k * scale, over the sum of the chosen scores if
// renormalised. Softmax: e_k / sum e; renormalised only the chosen logits
// enter.
//
// Balance of a sequence with n valid tokens: c_e pairs of expert e, f_e = E
// c_e / (topk n), P_e the mean of p_te (softmax, or the sigmoid over its
// row's sum), loss = sum f_e P_e, averaged over the sequences that have
// tokens.
//
// A row is one wave's: lane l holds the VPL experts l * VPL .. l * VPL + VPL -
// 1, so the first lane that holds the largest key also holds the lowest index.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <type_traits>

#include "common.h"

namespace xp {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kMaxTopk = 64;     // a lane per chosen expert
constexpr int kMaxGroups = 64;   // a lane per group
constexpr int kMaxGrouped = 1024;  // experts whose 64-bit keys four waves keep in LDS

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__hip_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void store_as(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_as(__hip_bfloat16* p, float v) { *p = __float2bfloat16(v); }
__device__ __forceinline__ void store_as(__half* p, float v) { *p = __float2half(v); }

// ---- reductions over the wave, the result in every lane ----
// Quad swaps, half-row and row mirrors (DPP), then the row and half swaps.
template <typename Op>
__device__ __forceinline__ uint32_t wave_reduce32(uint32_t v, Op op) {
  v = op(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xF, 0xF, false)));
  v = op(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4E, 0xF, 0xF, false)));
  v = op(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x141, 0xF, 0xF, false)));
  v = op(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x140, 0xF, 0xF, false)));
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = op(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return op(b[0], b[1]);
}

__device__ __forceinline__ float wave_sum(float v) {
  return __uint_as_float(wave_reduce32(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
__device__ __forceinline__ float wave_max(float v) {
  return __uint_as_float(wave_reduce32(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
__device__ __forceinline__ uint32_t wave_max_key(uint32_t v) {
  return wave_reduce32(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
__device__ __forceinline__ uint64_t wave_max_key(uint64_t v) {
  // The largest high word, then the largest low word among its holders.
  const uint32_t hi = wave_max_key(static_cast<uint32_t>(v >> 32));
  const uint32_t lo = wave_max_key(static_cast<uint32_t>(v >> 32) == hi ? static_cast<uint32_t>(v) : 0u);
  return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// ---- keys: unsigned numbers in the order of the values; 0: masked ----
__device__ __forceinline__ uint32_t order_key(float v) {
  if (!(v > -INFINITY)) return 0;  // NaN and -inf
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 counts as 0
  return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ uint64_t order_key(double v) {
  if (!(v > -static_cast<double>(INFINITY))) return 0;
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
  return b ^ (b >> 63 ? ~0ull : 0x8000000000000000ull);
}
__device__ __forceinline__ double key_value(uint64_t k) {
  return __longlong_as_double(static_cast<long long>(k ^ (k >> 63 ? 0x8000000000000000ull : ~0ull)));
}

// ---- a row's logits: masked ones as -inf ----
template <typename T, int VPL>
__device__ __forceinline__ void load_row(const T* __restrict__ row, int E, bool vec, float (&z)[VPL]) {
  constexpr int kBytes = VPL * static_cast<int>(sizeof(T));
  const int i0 = static_cast<int>(threadIdx.x & 63) * VPL;
  if (kBytes >= 4 && vec && i0 + VPL <= E) {
    T v[VPL];
    if constexpr (kBytes % 16 == 0) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i)
        reinterpret_cast<u32x4*>(v)[i] = reinterpret_cast<const u32x4*>(row + i0)[i];
    } else if constexpr (kBytes == 8) {
      *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(row + i0);
    } else if constexpr (kBytes == 4) {
      *reinterpret_cast<uint32_t*>(v) = *reinterpret_cast<const uint32_t*>(row + i0);
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) z[i] = to_float(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i) z[i] = i0 + i < E ? to_float(row[i0 + i]) : -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i) z[i] = z[i] > -INFINITY ? z[i] : -INFINITY;  // NaN is masked
}

// z - m for the row's maximum m: 0 at the maximum, an infinite one among them.
__device__ __forceinline__ float below(float z, float m) { return z == m ? 0.0f : z - m; }

// Terms t_i of the row's probabilities p_i = t_i / sum t, and the sum (0: the
// whole row is masked). Softmax: e^(z - m). Sigmoid: s e^-shift with shift =
// min(m, 0), so that a row of very negative logits keeps its ratios.
template <int VPL, bool SIGMOID>
__device__ __forceinline__ float row_terms(const float (&z)[VPL], float (&t)[VPL]) {
  float m = z[0];
#pragma unroll
  for (int i = 1; i < VPL; ++i) m = fmaxf(m, z[i]);
  m = wave_max(m);
  float sum = 0.0f;
  const float shift = fminf(m, 0.0f);
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    if constexpr (SIGMOID)
      t[i] = z[i] > 0.0f ? 1.0f / (1.0f + expf(-z[i])) : (z[i] > -INFINITY ? expf(z[i] - shift) / (1.0f + expf(z[i])) : 0.0f);
    else
      t[i] = z[i] > -INFINITY ? expf(below(z[i], m)) : 0.0f;
    sum += t[i];
  }
  return wave_sum(sum);
}

struct Pick {
  int topk, sigmoid, renorm, groups, keep;
  float scale;
  const float* bias;
};

// The round's winner: the largest key's lane and position. Returns its index
// (-1: every key is masked) and takes it out.
template <typename K, int VPL>
__device__ __forceinline__ int take_best(K (&key)[VPL]) {
  const int lane = threadIdx.x & 63;
  K best = key[0];
  int at = 0;
#pragma unroll
  for (int i = 1; i < VPL; ++i)
    if (key[i] > best) {
      best = key[i];
      at = i;
    }
  const K top = wave_max_key(best);
  if (top == 0) return -1;
  const int w = __ffsll(static_cast<long long>(__ballot(best == top))) - 1;
  const int v = __builtin_amdgcn_readlane(at, w);
  if (lane == w) {
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (i == v) key[i] = 0;
  }
  return w * VPL + v;
}

// Masks the keys of the groups that are not among the best `keep`. s_key: E
// keys of LDS for this wave.
template <typename K, int VPL>
__device__ __forceinline__ void keep_groups(K (&key)[VPL], int E, const Pick& pk, K* s_key) {
  const int lane = threadIdx.x & 63, size = E / pk.groups;
#pragma unroll
  for (int i = 0; i < VPL; ++i)
    if (lane * VPL + i < E) s_key[lane * VPL + i] = key[i];
  __builtin_amdgcn_wave_barrier();
  K worth[1] = {0};
  if (lane < pk.groups) {
    K a = 0, b = 0;  // the group's two largest keys
    for (int i = 0; i < size; ++i) {
      const K v = s_key[lane * size + i];
      if (v > a) {
        b = a;
        a = v;
      } else if (v > b) {
        b = v;
      }
    }
    worth[0] = a;
    if constexpr (sizeof(K) == 8) {
      if (b != 0) worth[0] = order_key(key_value(a) + key_value(b));
    }
  }
  __builtin_amdgcn_wave_barrier();
  uint64_t kept = 0;
  for (int g = 0; g < pk.keep; ++g) {
    const int best = take_best<K, 1>(worth);
    if (best < 0) break;
    kept |= 1ull << best;
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int e = lane * VPL + i;
    if (e < E && !(kept >> (e / size) & 1)) key[i] = 0;
  }
}

// The row's choice: lane k < topk gets the k-th id and its weight.
template <typename T, int VPL, bool WIDE>
__device__ __forceinline__ void choose_row(const T* __restrict__ row, const float (&z)[VPL], int E, const Pick& pk,
                                           void* s_key, int& id, float& weight) {
  using K = std::conditional_t<WIDE, uint64_t, uint32_t>;
  const int lane = threadIdx.x & 63;
  K key[VPL];
  if constexpr (WIDE) {
    double score[VPL], sum = 0.0;
    float m = z[0];
#pragma unroll
    for (int i = 1; i < VPL; ++i) m = fmaxf(m, z[i]);
    m = wave_max(m);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      if (!(z[i] > -INFINITY))
        score[i] = 0.0;
      else
        score[i] = pk.sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(z[i])))
                              : exp(z[i] == m ? 0.0 : static_cast<double>(z[i]) - static_cast<double>(m));
      sum += score[i];
    }
    sum = pk.sigmoid ? 1.0 : wave_sum(sum);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = lane * VPL + i;
      key[i] = z[i] > -INFINITY ? order_key(score[i] / sum + static_cast<double>(pk.bias[e])) : 0;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i) key[i] = order_key(z[i]);
  }
  if (pk.groups > 1) keep_groups<K, VPL>(key, E, pk, static_cast<K*>(s_key));
  id = -1;
  for (int k = 0; k < pk.topk; ++k) {
    const int best = take_best<K, VPL>(key);
    if (best < 0) break;
    if (lane == k) id = best;
  }
  // The chosen logits again (in the caches), one lane each.
  const float zc = id >= 0 ? to_float(row[id]) : -INFINITY;
  if (pk.sigmoid) {
    // In 64 bits; renormalised, the terms are s e^-shift (row_terms), so that
    // very negative logits keep their ratios.
    const double shift = pk.renorm ? fminf(wave_max(zc), 0.0f) : 0.0, zd = zc;
    const double s = id < 0 ? 0.0 : zc > 0.0f ? 1.0 / (1.0 + exp(-zd)) : exp(zd - shift) / (1.0 + exp(zd));
    const double all = pk.renorm ? wave_sum(s) : 1.0;
    weight = id >= 0 ? static_cast<float>(s / all * static_cast<double>(pk.scale)) : 0.0f;
    return;
  }
  float all;
  const float m = pk.renorm ? wave_max(zc) : 0.0f;
  float e;
  if (pk.renorm) {
    e = id >= 0 ? expf(below(zc, m)) : 0.0f;
    all = wave_sum(e);
  } else {
    float t[VPL];
    all = row_terms<VPL, false>(z, t);
    float top = z[0];
#pragma unroll
    for (int i = 1; i < VPL; ++i) top = fmaxf(top, z[i]);
    top = wave_max(top);
    e = id >= 0 ? expf(below(zc, top)) : 0.0f;
  }
  weight = id >= 0 ? e / all * pk.scale : 0.0f;
}

struct Rows {
  const void* logits;
  int64_t T, stride;
  int E;
  bool vec;
  const uint8_t* mask;
  const int32_t* offsets;  // sequences' first rows, num_seqs + 1, or null: all rows are one sequence
  int num_seqs;
};

// Rows [lo, hi) of sequence s, kept inside [0, T) whatever the offsets hold.
__device__ __forceinline__ void seq_range(const Rows& r, int s, int64_t& lo, int64_t& hi) {
  lo = 0;
  hi = r.T;
  if (r.offsets) {
    lo = r.offsets[s];
    hi = r.offsets[s + 1];
    lo = lo < 0 ? 0 : (lo < r.T ? lo : r.T);
    hi = hi < 0 ? 0 : (hi < r.T ? hi : r.T);
  }
}

template <typename T, int VPL, bool WIDE>
__global__ void __launch_bounds__(kThreads) choose_kernel(Rows r, Pick pk, float* __restrict__ weights,
                                                          int32_t* __restrict__ ids) {
  extern __shared__ __attribute__((aligned(16))) uint8_t s_raw[];  // [waves][E] keys where groups are used
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kWaves + wave;
  if (t >= r.T) return;
  int id = -1;
  float w = 0.0f;
  if (!r.mask || r.mask[t]) {
    const T* row = static_cast<const T*>(r.logits) + t * r.stride;
    float z[VPL];
    load_row<T, VPL>(row, r.E, r.vec, z);
    choose_row<T, VPL, WIDE>(row, z, r.E, pk, s_raw + static_cast<size_t>(wave) * r.E * (WIDE ? 8 : 4), id, w);
  }
  if (lane < pk.topk) {
    ids[t * pk.topk + lane] = id;
    weights[t * pk.topk + lane] = w;
  }
}

// Partial sums of one workgroup's rows of a sequence: [seq][part][E].
struct Partial {
  float* p;        // sums of the probabilities
  int32_t* c;      // counts
  int32_t* n;      // [seq][part] valid tokens
  int parts;
  double* loss;    // [seq]
};

// Workgroup (part j, sequence s): rows lo + 4 j + wave, + 4 parts, ... of the
// sequence; the sequence num_seqs stands for the rows outside all of them.
// CHOOSE: the choice is made here (else `given` holds it).
template <typename T, int VPL, bool SIGMOID, bool CHOOSE, bool WIDE>
__global__ void __launch_bounds__(kThreads) balance_kernel(Rows r, Pick pk, const void* __restrict__ given, int eb,
                                                           float* __restrict__ weights, int32_t* __restrict__ ids,
                                                           Partial out) {
  // [E] counts, then [waves][E] sums, in the same place as the waves' keys
  extern __shared__ __attribute__((aligned(16))) uint8_t s_raw[];
  int32_t* s_count = reinterpret_cast<int32_t*>(s_raw);
  uint8_t* s_rest = s_raw + ((static_cast<size_t>(r.E) * 4 + 15) & ~size_t(15));
  float* s_sum = reinterpret_cast<float*>(s_rest);
  __shared__ int s_valid[kWaves];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int s = blockIdx.y, j = blockIdx.x, E = r.E;
  if (s == r.num_seqs) {  // padding before and behind the sequences
    if constexpr (CHOOSE) {
      int64_t first = r.offsets[0], last = r.offsets[r.num_seqs];
      first = first < 0 ? 0 : (first < r.T ? first : r.T);
      last = last < first ? first : (last < r.T ? last : r.T);
      const int64_t n = (first + r.T - last) * pk.topk;
      for (int64_t i = static_cast<int64_t>(j) * kThreads + tid; i < n; i += static_cast<int64_t>(out.parts) * kThreads) {
        const int64_t at = i < first * pk.topk ? i : i + (last - first) * pk.topk;
        ids[at] = -1;
        weights[at] = 0.0f;
      }
    }
    return;
  }
  for (int i = tid; i < E; i += kThreads) s_count[i] = 0;
  __syncthreads();
  int64_t lo, hi;
  seq_range(r, s, lo, hi);
  float sum[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) sum[i] = 0.0f;
  int valid = 0;
  for (int64_t t = lo + static_cast<int64_t>(j) * kWaves + wave; t < hi; t += static_cast<int64_t>(out.parts) * kWaves) {
    const bool on = !r.mask || r.mask[t];
    int64_t id = -1;
    if (on) {
      const T* row = static_cast<const T*>(r.logits) + t * r.stride;
      float z[VPL], term[VPL];
      load_row<T, VPL>(row, E, r.vec, z);
      if constexpr (CHOOSE) {
        int mine;
        float w;
        choose_row<T, VPL, WIDE>(row, z, E, pk, s_rest + static_cast<size_t>(wave) * E * (WIDE ? 8 : 4), mine, w);
        if (lane < pk.topk) {
          ids[t * pk.topk + lane] = mine;
          weights[t * pk.topk + lane] = w;
        }
        id = mine;
      } else {
        if (lane < pk.topk) id = load_id(given, eb, t * pk.topk + lane);
      }
      if (id >= 0 && id < E) atomicAdd(&s_count[id], 1);
      const float all = row_terms<VPL, SIGMOID>(z, term);
      const float inv = all > 0.0f ? 1.0f / all : 0.0f;
#pragma unroll
      for (int i = 0; i < VPL; ++i) sum[i] += term[i] * inv;
      ++valid;
    } else if (CHOOSE) {
      if (lane < pk.topk) {
        ids[t * pk.topk + lane] = -1;
        weights[t * pk.topk + lane] = 0.0f;
      }
    }
  }
  __syncthreads();  // counts whole, and the keys' place is free
#pragma unroll
  for (int i = 0; i < VPL; ++i)
    if (lane * VPL + i < E) s_sum[wave * E + lane * VPL + i] = sum[i];
  if (lane == 0) s_valid[wave] = valid;
  __syncthreads();
  const int64_t part = static_cast<int64_t>(s) * out.parts + j;
  for (int i = tid; i < E; i += kThreads) {
    float a = s_sum[i];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) a += s_sum[w * E + i];
    out.p[part * E + i] = a;
    out.c[part * E + i] = s_count[i];
  }
  if (tid == 0) {
    int n = 0;
    for (int w = 0; w < kWaves; ++w) n += s_valid[w];
    out.n[part] = n;
  }
}

// Sum of v over the workgroup, in every thread of wave 0 at least.
__device__ __forceinline__ double block_sum(double v, double* s_tmp) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s_tmp[threadIdx.x >> 6] = v;
  __syncthreads();
  double all = 0.0;
  for (int w = 0; w < kWaves; ++w) all += s_tmp[w];
  return all;
}

// One sequence: its counts, valid tokens and loss from the partial sums, in 64 bits.
__global__ void __launch_bounds__(kThreads) balance_join_kernel(Partial in, int E, int topk,
                                                                int32_t* __restrict__ counts,
                                                                int32_t* __restrict__ tokens) {
  __shared__ double s_tmp[kWaves];
  const int s = blockIdx.x, tid = threadIdx.x;
  const int64_t base = static_cast<int64_t>(s) * in.parts;
  double n = 0.0;
  for (int j = tid; j < in.parts; j += kThreads) n += in.n[base + j];
  n = block_sum(n, s_tmp);
  double loss = 0.0;
  for (int e = tid; e < E; e += kThreads) {
    double p = 0.0;
    int32_t c = 0;
    for (int j = 0; j < in.parts; ++j) {
      p += in.p[(base + j) * E + e];
      c += in.c[(base + j) * E + e];
    }
    counts[static_cast<int64_t>(s) * E + e] = c;
    loss += p * c;
  }
  loss = block_sum(loss, s_tmp);
  if (tid == 0) {
    tokens[s] = static_cast<int32_t>(n);
    in.loss[s] = n > 0.0 ? loss * E / (n * n * topk) : 0.0;
  }
}

// The mean over the sequences with tokens; tokens[num_seqs] = their number.
__global__ void __launch_bounds__(kThreads) balance_mean_kernel(Partial in, int num_seqs, int32_t* __restrict__ tokens,
                                                                float* __restrict__ loss) {
  __shared__ double s_tmp[kWaves];
  double a = 0.0, used = 0.0;
  for (int s = threadIdx.x; s < num_seqs; s += kThreads) {
    a += in.loss[s];
    used += tokens[s] > 0 ? 1.0 : 0.0;
  }
  a = block_sum(a, s_tmp);
  used = block_sum(used, s_tmp);
  if (threadIdx.x == 0) {
    tokens[num_seqs] = static_cast<int32_t>(used);
    *loss = static_cast<float>(used > 0.0 ? a / used : 0.0);
  }
}

struct Back {
  const void* ids;
  int eb;
  const float* grad_weights;  // null: none
  const int32_t* counts;      // null: no loss
  const int32_t* tokens;
  const float* grad_loss;
};

// d/dz of a row. With G_i the gradient by the probability p_i (the loss's
// g f_i / (n B), and scale g_k at the chosen experts of a softmax that is not
// renormalised), dz_i = p_i (G_i - sum G p), times 1 - s_i for the sigmoid.
// Renormalised weights w_k = scale w'_k depend on the chosen logits alone: dz_k
// += scale w'_k (g_k - sum g w'), times 1 - s_k; the sigmoid's own: dz_k +=
// scale g_k s_k (1 - s_k).
template <typename T, int VPL, bool SIGMOID>
__global__ void __launch_bounds__(kThreads) backward_kernel(Rows r, Pick pk, Back b, T* __restrict__ grad) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, E = r.E;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kWaves + wave;
  if (t >= r.T) return;
  // The row's sequence: the last one that starts at or before it, and ends behind it.
  int s = 0;
  bool on = !r.mask || r.mask[t];
  if (on && r.offsets) {
    int a = 0, z = r.num_seqs;
    while (z - a > 1) {
      const int m = (a + z) >> 1;
      if (r.offsets[m] <= t)
        a = m;
      else
        z = m;
    }
    s = a;
    on = r.offsets[s] <= t && t < r.offsets[s + 1];
  }
  float z[VPL], p[VPL], dz[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) dz[i] = 0.0f;
  if (on) {
    const T* row = static_cast<const T*>(r.logits) + t * r.stride;
    load_row<T, VPL>(row, E, r.vec, z);
    const float all = row_terms<VPL, SIGMOID>(z, p);
    const float inv = all > 0.0f ? 1.0f / all : 0.0f;
    float G[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      p[i] *= inv;
      G[i] = 0.0f;
    }
    if (b.counts) {
      const double n = b.tokens[s];
      const float k = n > 0.0 ? static_cast<float>(static_cast<double>(*b.grad_loss) * E /
                                                   (n * n * pk.topk * b.tokens[r.num_seqs]))
                              : 0.0f;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (lane * VPL + i < E) G[i] = k * static_cast<float>(b.counts[static_cast<int64_t>(s) * E + lane * VPL + i]);
    }
    int id = -1;
    float direct = 0.0f;
    if (b.grad_weights) {
      float g = 0.0f;
      if (lane < pk.topk) {
        const int64_t e = load_id(b.ids, b.eb, t * pk.topk + lane);
        id = e >= 0 && e < E ? static_cast<int>(e) : -1;
        g = id >= 0 ? b.grad_weights[t * pk.topk + lane] * pk.scale : 0.0f;
      }
      const float zc = id >= 0 ? to_float(row[id]) : -INFINITY;
      if (pk.renorm) {
        // w' of the chosen: the terms by the largest chosen logit, as in the choice.
        const float m = wave_max(zc);
        float e = 0.0f, slope = 1.0f;
        if (id >= 0) {
          if (SIGMOID) {
            const float shift = fminf(m, 0.0f), ez = expf(-fabsf(zc));
            e = zc > 0.0f ? 1.0f / (1.0f + ez) : expf(zc - shift) / (1.0f + ez);
            slope = zc > 0.0f ? ez / (1.0f + ez) : 1.0f / (1.0f + ez);
          } else {
            e = expf(below(zc, m));
          }
        }
        const float sum = wave_sum(e);
        const float w = sum > 0.0f ? e / sum : 0.0f;
        direct = w * slope * (g - wave_sum(g * w));
      } else if (SIGMOID) {
        const float ez = expf(-fabsf(zc));
        direct = id >= 0 ? g * ez / ((1.0f + ez) * (1.0f + ez)) : 0.0f;
      }
      if (!pk.renorm && !SIGMOID) {
        for (int k = 0; k < pk.topk; ++k) {
          const int e = __builtin_amdgcn_readlane(id, k);
          const float v = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(g), k));
#pragma unroll
          for (int i = 0; i < VPL; ++i)
            if (e == lane * VPL + i) G[i] += v;
        }
      }
    }
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) dot += G[i] * p[i];
    dot = wave_sum(dot);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      dz[i] = p[i] * (G[i] - dot);
      if (SIGMOID && z[i] > -INFINITY) dz[i] *= 1.0f / (1.0f + expf(z[i]));
    }
    if (b.grad_weights && (pk.renorm || SIGMOID)) {
      for (int k = 0; k < pk.topk; ++k) {
        const int e = __builtin_amdgcn_readlane(id, k);
        const float v = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(direct), k));
#pragma unroll
        for (int i = 0; i < VPL; ++i)
          if (e == lane * VPL + i) dz[i] += v;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i)
    if (lane * VPL + i < E) store_as(grad + t * E + lane * VPL + i, dz[i]);
}

// ---- host side ----

struct Call {
  const char* what;
  const void* logits;
  int dtype;
  int64_t T, E, stride;
  const uint8_t* mask;
  const int32_t* offsets;
  int64_t num_seqs;
};

int check_rows(const Call& c) {
  XP_REQUIRE(c.dtype >= XP_FLOAT32 && c.dtype <= XP_FLOAT16, "%s: unknown logits type %d", c.what, c.dtype);
  XP_REQUIRE(c.T >= 0 && c.T <= INT32_MAX && c.E >= 1 && c.E <= XP_MAX_EXPERTS, "%s: T=%lld, E=%lld (at most %d experts)",
             c.what, (long long)c.T, (long long)c.E, XP_MAX_EXPERTS);
  XP_REQUIRE(c.stride >= c.E || c.T <= 1, "%s: rows of %lld logits are %lld apart", c.what, (long long)c.E,
             (long long)c.stride);
  XP_REQUIRE(c.num_seqs >= 1 && c.num_seqs <= 65534 && (c.offsets || c.num_seqs == 1),
             "%s: %lld sequences (1 to 65534)", c.what, (long long)c.num_seqs);
  XP_REQUIRE(c.T == 0 || c.logits, "%s: null logits", c.what);
  return XP_OK;
}

int check_pick(const char* what, int64_t E, int64_t topk, int scoring, int64_t groups, int64_t keep, double scale) {
  XP_REQUIRE(topk >= 1 && topk <= kMaxTopk && topk <= E, "%s: topk=%lld of %lld experts (at most %d)", what,
             (long long)topk, (long long)E, kMaxTopk);
  XP_REQUIRE(scoring == XP_SCORE_SOFTMAX || scoring == XP_SCORE_SIGMOID, "%s: unknown scoring %d", what, scoring);
  XP_REQUIRE(groups >= 1 && groups <= kMaxGroups && E % groups == 0 && keep >= 1 && keep <= groups &&
                 topk <= E / groups * keep,
             "%s: %lld of %lld groups (at most %d, of equal size) for the %lld best of %lld experts", what,
             (long long)keep, (long long)groups, kMaxGroups, (long long)topk, (long long)E);
  XP_REQUIRE(groups == 1 || E <= kMaxGrouped, "%s: groups over %lld experts (at most %d)", what, (long long)E,
             kMaxGrouped);
  XP_REQUIRE(scale == scale && scale - scale == 0.0, "%s: scale must be finite", what);
  return XP_OK;
}

size_t elem_bytes(int dtype) { return dtype == XP_FLOAT32 ? 4 : 2; }

// The experts a lane holds: the least power of two that covers E.
int values_per_lane(int64_t E) {
  int v = 1;
  while (64 * v < E) v *= 2;
  return v;
}

Rows rows_of(const Call& c) {
  const size_t eb = elem_bytes(c.dtype), chunk = std::min<size_t>(16, values_per_lane(c.E) * eb);
  Rows r{c.logits, c.T, c.stride, static_cast<int>(c.E), false, c.mask, c.offsets, static_cast<int>(c.num_seqs)};
  r.vec = reinterpret_cast<uintptr_t>(c.logits) % chunk == 0 && c.stride * eb % chunk == 0;
  return r;
}

template <int N>
using Int = std::integral_constant<int, N>;

// f(T{}, Int<VPL>{}) for the logits' type and the experts per lane.
template <typename F>
void dispatch(int dtype, int vpl, F&& f) {
  auto by_type = [&](auto v) {
    if (dtype == XP_FLOAT32)
      f(float{}, v);
    else if (dtype == XP_BFLOAT16)
      f(__hip_bfloat16{}, v);
    else
      f(__half{}, v);
  };
  switch (vpl) {
    case 1: return by_type(Int<1>{});
    case 2: return by_type(Int<2>{});
    case 4: return by_type(Int<4>{});
    case 8: return by_type(Int<8>{});
    case 16: return by_type(Int<16>{});
    default: return by_type(Int<32>{});
  }
}

// Workgroups that share a sequence.
int balance_parts(int64_t T, int64_t num_seqs) {
  const int64_t per = (T + num_seqs - 1) / num_seqs;
  int64_t parts = (per + 4 * kWaves - 1) / (4 * kWaves);  // four rows a wave at least
  parts = std::min<int64_t>(parts, std::max<int64_t>(1, 512 / num_seqs));
  return static_cast<int>(std::max<int64_t>(parts, 1));
}

int64_t align256(int64_t n) { return (n + 255) & ~int64_t(255); }

int64_t balance_layout(int64_t T, int64_t E, int64_t num_seqs, Partial* p, uint8_t* base) {
  const int64_t parts = balance_parts(T, num_seqs), n = parts * num_seqs;
  const int64_t sz[4] = {align256(n * E * 4), align256(n * E * 4), align256(n * 4), align256(num_seqs * 8)};
  if (p) {
    p->parts = static_cast<int>(parts);
    p->p = reinterpret_cast<float*>(base);
    p->c = reinterpret_cast<int32_t*>(base + sz[0]);
    p->n = reinterpret_cast<int32_t*>(base + sz[0] + sz[1]);
    p->loss = reinterpret_cast<double*>(base + sz[0] + sz[1] + sz[2]);
  }
  return sz[0] + sz[1] + sz[2] + sz[3];
}

int launch_balance(const Call& c, const Pick& pk, bool choose, const void* given, int eb, float* weights, int32_t* ids,
                   void* work, int32_t* counts, int32_t* tokens, float* loss, void* stream) {
  const hipStream_t st = as_stream(stream);
  Partial part{};
  balance_layout(c.T, c.E, c.num_seqs, &part, static_cast<uint8_t*>(work));
  const bool wide = choose && pk.bias;
  const size_t keys = choose && pk.groups > 1 ? static_cast<size_t>(kWaves) * c.E * (wide ? 8 : 4) : 0;
  const size_t lds = ((c.E * 4 + 15) & ~size_t(15)) + std::max(keys, static_cast<size_t>(kWaves) * c.E * 4);
  const dim3 grid(static_cast<unsigned>(part.parts), static_cast<unsigned>(c.num_seqs + (choose && c.offsets ? 1 : 0)));
  const Rows r = rows_of(c);
  dispatch(c.dtype, values_per_lane(c.E), [&](auto type, auto v) {
    using T = decltype(type);
    constexpr int V = decltype(v)::value;
    auto go = [&](auto* kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(kThreads), lds, st, r, pk, given, eb, weights, ids, part);
    };
    if (!choose)
      pk.sigmoid ? go(balance_kernel<T, V, true, false, false>) : go(balance_kernel<T, V, false, false, false>);
    else if (wide)
      pk.sigmoid ? go(balance_kernel<T, V, true, true, true>) : go(balance_kernel<T, V, false, true, true>);
    else
      pk.sigmoid ? go(balance_kernel<T, V, true, true, false>) : go(balance_kernel<T, V, false, true, false>);
  });
  if (int rc = check_launch("balance_kernel")) return rc;
  hipLaunchKernelGGL(balance_join_kernel, dim3(static_cast<unsigned>(c.num_seqs)), dim3(kThreads), 0, st, part,
                     static_cast<int>(c.E), pk.topk, counts, tokens);
  if (int rc = check_launch("balance_join_kernel")) return rc;
  hipLaunchKernelGGL(balance_mean_kernel, dim3(1), dim3(kThreads), 0, st, part, static_cast<int>(c.num_seqs), tokens,
                     loss);
  return check_launch("balance_mean_kernel");
}

}  // namespace
}  // namespace xp

using namespace xp;

extern "C" {

int xp_router_choose(const void* logits, int dtype, int64_t T, int64_t E, int64_t row_stride, int64_t topk, int scoring,
                     int renormalize, const float* bias, int64_t groups, int64_t topk_groups, double scale,
                     const uint8_t* mask, float* weights, int32_t* ids, void* stream) {
  const char* what = "xp_router_choose";
  const Call c{what, logits, dtype, T, E, row_stride, mask, nullptr, 1};
  if (int rc = check_rows(c)) return rc;
  if (int rc = check_pick(what, E, topk, scoring, groups, topk_groups, scale)) return rc;
  if (T == 0) return XP_OK;
  XP_REQUIRE(weights && ids, "%s: null output", what);
  const Pick pk{static_cast<int>(topk), scoring == XP_SCORE_SIGMOID, renormalize != 0, static_cast<int>(groups),
                static_cast<int>(topk_groups), static_cast<float>(scale), bias};
  const Rows r = rows_of(c);
  const size_t lds = groups > 1 ? static_cast<size_t>(kWaves) * E * (bias ? 8 : 4) : 0;
  const dim3 grid(static_cast<unsigned>((T + kWaves - 1) / kWaves));
  dispatch(dtype, values_per_lane(E), [&](auto type, auto v) {
    using L = decltype(type);
    constexpr int V = decltype(v)::value;
    auto* kernel = bias ? choose_kernel<L, V, true> : choose_kernel<L, V, false>;
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), lds, as_stream(stream), r, pk, weights, ids);
  });
  return check_launch("choose_kernel");
}

int64_t xp_router_workspace_bytes(int64_t T, int64_t E, int64_t num_seqs) {
  if (T < 0 || E < 1 || num_seqs < 1) return 0;
  return balance_layout(T, E, num_seqs, nullptr, nullptr);
}

int xp_router_balance(const void* logits, int dtype, int64_t T, int64_t E, int64_t row_stride, int64_t topk, int scoring,
                      const void* topk_ids, int topk_elem_bytes, const uint8_t* mask, const int32_t* seq_offsets,
                      int64_t num_seqs, void* work, int64_t work_bytes, int32_t* counts, int32_t* tokens, float* loss,
                      void* stream) {
  const char* what = "xp_router_balance";
  const Call c{what, logits, dtype, T, E, row_stride, mask, seq_offsets, num_seqs};
  if (int rc = check_rows(c)) return rc;
  // Any number of the same expert may stand in a given choice: topk is bounded by the lanes alone.
  XP_REQUIRE(topk >= 1 && topk <= kMaxTopk, "%s: topk=%lld (at most %d)", what, (long long)topk, kMaxTopk);
  XP_REQUIRE(scoring == XP_SCORE_SOFTMAX || scoring == XP_SCORE_SIGMOID, "%s: unknown scoring %d", what, scoring);
  XP_REQUIRE(topk_elem_bytes == 4 || topk_elem_bytes == 8, "%s: id size %d", what, topk_elem_bytes);
  XP_REQUIRE((T == 0 || topk_ids) && counts && tokens && loss, "%s: null argument", what);
  XP_REQUIRE(work && (reinterpret_cast<uintptr_t>(work) & 255) == 0 &&
                 work_bytes >= xp_router_workspace_bytes(T, E, num_seqs),
             "%s: the workspace must be 256-byte aligned and of %lld B", what,
             (long long)xp_router_workspace_bytes(T, E, num_seqs));
  const Pick pk{static_cast<int>(topk), scoring == XP_SCORE_SIGMOID, 0, 1, 1, 1.0f, nullptr};
  return launch_balance(c, pk, false, topk_ids, topk_elem_bytes, nullptr, nullptr, work, counts, tokens, loss, stream);
}

int xp_router_choose_balance(const void* logits, int dtype, int64_t T, int64_t E, int64_t row_stride, int64_t topk,
                             int scoring, int renormalize, const float* bias, int64_t groups, int64_t topk_groups,
                             double scale, const uint8_t* mask, const int32_t* seq_offsets, int64_t num_seqs,
                             float* weights, int32_t* ids, void* work, int64_t work_bytes, int32_t* counts,
                             int32_t* tokens, float* loss, void* stream) {
  const char* what = "xp_router_choose_balance";
  const Call c{what, logits, dtype, T, E, row_stride, mask, seq_offsets, num_seqs};
  if (int rc = check_rows(c)) return rc;
  if (int rc = check_pick(what, E, topk, scoring, groups, topk_groups, scale)) return rc;
  XP_REQUIRE((T == 0 || (weights && ids)) && counts && tokens && loss, "%s: null argument", what);
  XP_REQUIRE(work && (reinterpret_cast<uintptr_t>(work) & 255) == 0 &&
                 work_bytes >= xp_router_workspace_bytes(T, E, num_seqs),
             "%s: the workspace must be 256-byte aligned and of %lld B", what,
             (long long)xp_router_workspace_bytes(T, E, num_seqs));
  const Pick pk{static_cast<int>(topk), scoring == XP_SCORE_SIGMOID, renormalize != 0, static_cast<int>(groups),
                static_cast<int>(topk_groups), static_cast<float>(scale), bias};
  return launch_balance(c, pk, true, nullptr, 4, weights, ids, work, counts, tokens, loss, stream);
}

int xp_router_backward(const void* logits, int dtype, int64_t T, int64_t E, int64_t row_stride, int64_t topk,
                       int scoring, int renormalize, double scale, const uint8_t* mask, const int32_t* seq_offsets,
                       int64_t num_seqs, const void* topk_ids, int topk_elem_bytes, const float* grad_weights,
                       const int32_t* counts, const int32_t* tokens, const float* grad_loss, void* grad,
                       void* stream) {
  const char* what = "xp_router_backward";
  const Call c{what, logits, dtype, T, E, row_stride, mask, seq_offsets, num_seqs};
  if (int rc = check_rows(c)) return rc;
  XP_REQUIRE(topk >= 1 && topk <= kMaxTopk, "%s: topk=%lld (at most %d)", what, (long long)topk, kMaxTopk);
  XP_REQUIRE(scoring == XP_SCORE_SOFTMAX || scoring == XP_SCORE_SIGMOID, "%s: unknown scoring %d", what, scoring);
  XP_REQUIRE(topk_elem_bytes == 4 || topk_elem_bytes == 8, "%s: id size %d", what, topk_elem_bytes);
  XP_REQUIRE(grad_weights == nullptr || topk_ids, "%s: the weights' gradient needs the ids", what);
  XP_REQUIRE((counts == nullptr) == (grad_loss == nullptr) && (counts == nullptr) == (tokens == nullptr),
             "%s: the loss's gradient needs counts, tokens and grad_loss", what);
  XP_REQUIRE(scale == scale && scale - scale == 0.0, "%s: scale must be finite", what);
  if (T == 0) return XP_OK;
  XP_REQUIRE(grad, "%s: null gradient", what);
  const Pick pk{static_cast<int>(topk), scoring == XP_SCORE_SIGMOID, renormalize != 0, 1, 1, static_cast<float>(scale),
                nullptr};
  const Back b{topk_ids, topk_elem_bytes, grad_weights, counts, tokens, grad_loss};
  const Rows r = rows_of(c);
  const dim3 grid(static_cast<unsigned>((T + kWaves - 1) / kWaves));
  dispatch(dtype, values_per_lane(E), [&](auto type, auto v) {
    using L = decltype(type);
    constexpr int V = decltype(v)::value;
    auto* kernel = pk.sigmoid ? backward_kernel<L, V, true> : backward_kernel<L, V, false>;
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, as_stream(stream), r, pk, b, static_cast<L*>(grad));
  });
  return check_launch("backward_kernel");
}

}  // extern "C"

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
// Two forms. Up to 512 experts and 16 choices without bias and groups, a row is
// 16 lanes' (four rows a wave): lane l holds the VPL experts l * VPL .. l * VPL
// + VPL - 1, and the choice is a merge of sorted lists, with no step that waits
// on the one before it for long. Otherwise a row is a wave's, and the choice a
// round per expert: the largest key of all lanes, its first holder, and that
// key taken out. 32768 tokens of 256 experts, top-8, bf16, choice and loss: 18 us
// by the first form, 62 by the second; their backward 13.5 and 29 (other sizes at
// narrow_rows). Bound there by VALU instructions (1.1 and 2.6 TB/s); 4096 tokens
// in 8 groups with a bias, 13 us, by the rounds; below some hundred tokens by a
// launch's latency (2.7 us).
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <cfloat>
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
// A double's halves moved by a DPP control, or swapped between rows (16) or halves (32) of the wave.
template <int CTRL>
__device__ __forceinline__ double move_lanes(double v) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v));
  const uint64_t lo = static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(b), CTRL, 0xF, 0xF, false));
  const uint64_t hi = static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(b >> 32), CTRL, 0xF, 0xF, false));
  return __longlong_as_double(static_cast<long long>(hi << 32 | lo));
}
template <int ROWS, typename Op>
__device__ __forceinline__ double across(double v, Op op) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v));
  const uint32_t l = static_cast<uint32_t>(b), h = static_cast<uint32_t>(b >> 32);
  uint64_t x, y;
  if constexpr (ROWS == 16) {
    const auto lo = __builtin_amdgcn_permlane16_swap(l, l, false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap(h, h, false, false);
    x = static_cast<uint64_t>(hi[0]) << 32 | lo[0];
    y = static_cast<uint64_t>(hi[1]) << 32 | lo[1];
  } else {
    const auto lo = __builtin_amdgcn_permlane32_swap(l, l, false, false);
    const auto hi = __builtin_amdgcn_permlane32_swap(h, h, false, false);
    x = static_cast<uint64_t>(hi[0]) << 32 | lo[0];
    y = static_cast<uint64_t>(hi[1]) << 32 | lo[1];
  }
  return op(__longlong_as_double(static_cast<long long>(x)), __longlong_as_double(static_cast<long long>(y)));
}
template <typename Op>
__device__ __forceinline__ double wave_reduce64(double v, Op op) {
  v = op(v, move_lanes<0xB1>(v));
  v = op(v, move_lanes<0x4E>(v));
  v = op(v, move_lanes<0x141>(v));
  v = op(v, move_lanes<0x140>(v));
  v = across<16>(v, op);
  return across<32>(v, op);
}
__device__ __forceinline__ double wave_max_key(double v) {
  return wave_reduce64(v, [](double a, double b) { return __builtin_fmax(a, b); });
}
__device__ __forceinline__ double wave_sum(double v) {
  return wave_reduce64(v, [](double a, double b) { return a + b; });
}

// ---- keys ----
// A logit's key is an unsigned number in its order (0: masked); a score with a
// bias is its own key in 64 bits (-inf: masked), whose maximum is one
// instruction where that of 64-bit integers is five.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (!(v > -INFINITY)) return 0;  // NaN and -inf
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 counts as 0
  return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
template <typename K>
__device__ __forceinline__ K masked_key() {
  if constexpr (std::is_same_v<K, double>)
    return -static_cast<double>(INFINITY);
  else
    return 0;
}
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t smaller(uint32_t a, uint32_t b) { return a > b ? b : a; }
__device__ __forceinline__ double larger(double a, double b) { return __builtin_fmax(a, b); }
__device__ __forceinline__ double smaller(double a, double b) { return __builtin_fmin(a, b); }

// ---- a row's logits: masked ones as -inf ----
// LANES lanes hold a row, VPL consecutive experts each.
template <typename T, int VPL, int LANES>
__device__ __forceinline__ void load_part(const T* __restrict__ row, int E, bool vec, float (&z)[VPL]) {
  constexpr int kBytes = VPL * static_cast<int>(sizeof(T));
  const int i0 = static_cast<int>(threadIdx.x & (LANES - 1)) * VPL;
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

// The round's winner: the first lane that holds the largest key, and there the
// first position. Returns its index (-1: every key is masked) and takes it out.
template <typename K, int VPL>
__device__ __forceinline__ int take_best(K (&key)[VPL]) {
  const int lane = threadIdx.x & 63;
  K best = key[0];
#pragma unroll
  for (int i = 1; i < VPL; ++i) best = larger(best, key[i]);
  const K top = wave_max_key(best);
  if (top == masked_key<K>()) return -1;
  const int w = __ffsll(static_cast<long long>(__ballot(best == top))) - 1;
  int at = VPL - 1;
#pragma unroll
  for (int i = VPL - 2; i >= 0; --i) at = key[i] == top ? i : at;
  const int v = __builtin_amdgcn_readlane(at, w);
#pragma unroll
  for (int i = 0; i < VPL; ++i) key[i] = lane == w && i == v ? masked_key<K>() : key[i];
  return w * VPL + v;
}

// A group's two largest keys, a >= b.
template <typename K>
__device__ __forceinline__ void take_two(K& a, K& b, K v) {
  b = larger(b, smaller(a, v));
  a = larger(a, v);
}
// What a group counts: its largest key, or with a bias the sum of the two largest.
template <typename K>
__device__ __forceinline__ K group_worth(K a, K b) {
  if constexpr (std::is_same_v<K, double>)
    return b > masked_key<K>() ? a + b : a;
  else
    return a;
}

// Masks the keys of the groups that are not among the best `keep`. A group of
// 2^n whole lanes (256 experts in 8 groups: 8 lanes) is summed up by steps over
// its lanes; others through s_key, E keys of LDS for this wave, by a lane each.
template <typename K, int VPL>
__device__ __forceinline__ void keep_groups(K (&key)[VPL], int E, const Pick& pk, K* s_key) {
  const int lane = threadIdx.x & 63, size = E / pk.groups;
  const int span = size / VPL;  // lanes of a group
  const bool lanes = size % VPL == 0 && (span & (span - 1)) == 0;
  K worth[1] = {masked_key<K>()};
  int group_of = lane;  // the group that this lane answers for
  if (lanes) {
    K a = key[0], b = masked_key<K>();
#pragma unroll
    for (int i = 1; i < VPL; ++i) take_two(a, b, key[i]);
    for (int d = 1; d < span; d <<= 1) {
      const K oa = __shfl_xor(a, d, 64), ob = __shfl_xor(b, d, 64);
      take_two(a, b, oa);
      b = larger(b, ob);
    }
    if (lane % span == 0 && lane * VPL < E) worth[0] = group_worth(a, b);
    group_of = lane / span;
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (lane * VPL + i < E) s_key[lane * VPL + i] = key[i];
    __builtin_amdgcn_wave_barrier();
    if (lane < pk.groups) {
      K a = masked_key<K>(), b = masked_key<K>();
      for (int i = 0; i < size; ++i) take_two(a, b, s_key[lane * size + i]);
      worth[0] = group_worth(a, b);
    }
    __builtin_amdgcn_wave_barrier();
  }
  uint64_t kept = 0;
  for (int g = 0; g < pk.keep; ++g) {
    const int best = take_best<K, 1>(worth);
    if (best < 0) break;
    kept |= 1ull << __builtin_amdgcn_readlane(group_of, best);
  }
  if (lanes) {
    const bool mine = kept >> (group_of & 63) & 1;
#pragma unroll
    for (int i = 0; i < VPL; ++i) key[i] = mine ? key[i] : masked_key<K>();
    return;
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int e = lane * VPL + i;
    if (e < E && !(kept >> (e / size) & 1)) key[i] = masked_key<K>();
  }
}

// The row's choice: lane k < topk gets the k-th id and its weight.
template <typename T, int VPL, bool WIDE>
__device__ __forceinline__ void choose_row(const T* __restrict__ row, const float (&z)[VPL], int E, const Pick& pk,
                                           void* s_key, int& id, float& weight) {
  using K = std::conditional_t<WIDE, double, uint32_t>;
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
    const double inv = pk.sigmoid ? 1.0 : 1.0 / wave_sum(sum);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = lane * VPL + i;
      const double k = z[i] > -INFINITY ? score[i] * inv + static_cast<double>(pk.bias[e]) : masked_key<double>();
      key[i] = k > masked_key<double>() ? k : masked_key<double>();  // (a bias may be NaN)
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
    load_part<T, VPL, 64>(row, r.E, r.vec, z);
    choose_row<T, VPL, WIDE>(row, z, r.E, pk, s_raw + static_cast<size_t>(wave) * r.E * (WIDE ? 8 : 4), id, w);
  }
  if (lane < pk.topk) {
    ids[t * pk.topk + lane] = id;
    weights[t * pk.topk + lane] = w;
  }
}

// What the workgroups hand to the join.
struct Partial {
  uint2* pc;       // [seq][part][E]: sum of the probabilities (fp32 bits), count
  int32_t* n;      // [seq][part] valid tokens
  int parts;
  double* loss;    // [seq][expert block]: the block's part of the sequence's loss (-1: no tokens)
  int32_t* done;   // join workgroups that are done
};

// A workgroup's sums ([waves][pitch] in LDS), counts and valid tokens.
__device__ __forceinline__ void store_partial(const Partial& out, int s, int j, int E, const int32_t* s_count,
                                              const float* s_sum, int pitch, const int* s_valid) {
  const int tid = threadIdx.x;
  const int64_t part = static_cast<int64_t>(s) * out.parts + j;
  for (int i = tid; i < E; i += kThreads) {
    float a = s_sum[i];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) a += s_sum[w * pitch + i];
    out.pc[part * E + i] = make_uint2(__float_as_uint(a), static_cast<uint32_t>(s_count[i]));
  }
  if (tid == 0) {
    int n = 0;
    for (int w = 0; w < kWaves; ++w) n += s_valid[w];
    out.n[part] = n;
  }
}

// The rows before and behind the sequences: no choice. Part j of `parts`.
__device__ __forceinline__ void mark_padding(const Rows& r, int topk, float* weights, int32_t* ids, int j, int parts) {
  int64_t first = r.offsets[0], last = r.offsets[r.num_seqs];
  first = first < 0 ? 0 : (first < r.T ? first : r.T);
  last = last < first ? first : (last < r.T ? last : r.T);
  const int64_t n = (first + r.T - last) * topk;
  for (int64_t i = static_cast<int64_t>(j) * kThreads + threadIdx.x; i < n; i += static_cast<int64_t>(parts) * kThreads) {
    const int64_t at = i < first * topk ? i : i + (last - first) * topk;
    ids[at] = -1;
    weights[at] = 0.0f;
  }
}

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
  if (s == 0 && j == 0 && tid == 0) *out.done = 0;
  if (s == r.num_seqs) {
    if constexpr (CHOOSE) mark_padding(r, pk.topk, weights, ids, j, out.parts);
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
      load_part<T, VPL, 64>(row, E, r.vec, z);
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
  store_partial(out, s, j, E, s_count, s_sum, E, s_valid);
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

constexpr int kJoinExperts = 16;  // experts of a join workgroup (128 bytes of a part's row)

// Workgroup (expert block, sequence): the block's counts and its part of the
// loss, from the partial sums, in 64 bits. The workgroup that is done last
// adds the parts up, in the order of sequences and blocks whoever it is.
__global__ void __launch_bounds__(kThreads) balance_join_kernel(Partial in, int E, int topk, int num_seqs,
                                                                int32_t* __restrict__ counts,
                                                                int32_t* __restrict__ tokens,
                                                                float* __restrict__ loss) {
  constexpr int kAcross = kThreads / kJoinExperts;  // parts summed side by side
  __shared__ double s_tmp[kWaves];
  __shared__ double s_p[kAcross][kJoinExperts];
  __shared__ int s_c[kAcross][kJoinExperts];
  __shared__ int s_last;
  const int s = blockIdx.y, tid = threadIdx.x;
  const int x = tid % kJoinExperts, y = tid / kJoinExperts, e = blockIdx.x * kJoinExperts + x;
  const int64_t base = static_cast<int64_t>(s) * in.parts;
  double n = 0.0, p = 0.0;
  int c = 0;
  if (e < E) {
#pragma unroll 8
    for (int j = y; j < in.parts; j += kAcross) {
      const uint2 v = in.pc[(base + j) * E + e];
      p += __uint_as_float(v.x);
      c += static_cast<int>(v.y);
    }
  }
  for (int j = tid; j < in.parts; j += kThreads) n += in.n[base + j];
  s_p[y][x] = p;
  s_c[y][x] = c;
  n = block_sum(n, s_tmp);
  double part = 0.0;
  if (tid < kJoinExperts && e < E) {
    for (int i = 1; i < kAcross; ++i) {
      p += s_p[i][x];
      c += s_c[i][x];
    }
    counts[static_cast<int64_t>(s) * E + e] = c;
    part = p * c;
  }
  part = block_sum(part, s_tmp);
  if (tid == 0) {
    if (blockIdx.x == 0) tokens[s] = static_cast<int32_t>(n);
    in.loss[static_cast<int64_t>(s) * gridDim.x + blockIdx.x] = n > 0.0 ? part * E / (n * n * topk) : -1.0;
    const int total = static_cast<int>(gridDim.x * gridDim.y);
    s_last = __hip_atomic_fetch_add(in.done, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == total - 1;
  }
  __syncthreads();
  if (!s_last) return;
  double a = 0.0, used = 0.0;
  const int64_t all = static_cast<int64_t>(num_seqs) * gridDim.x;
  for (int64_t i = tid; i < all; i += kThreads) {
    const double v = __hip_atomic_load(in.loss + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (v < 0.0) continue;
    a += v;
    used += i % gridDim.x == 0 ? 1.0 : 0.0;
  }
  a = block_sum(a, s_tmp);
  used = block_sum(used, s_tmp);
  if (tid == 0) {
    tokens[num_seqs] = static_cast<int32_t>(used);
    *loss = static_cast<float>(used > 0.0 ? a / used : 0.0);
  }
}

// ---- rows of 16 lanes ----

constexpr int kRowLanes = 16;
constexpr int kRowsPerWave = 64 / kRowLanes;
constexpr int kBlockRows = kWaves * kRowsPerWave;
constexpr int kNarrowExperts = 512;  // experts of a row of 16 lanes, at most (32 a lane)
constexpr int kNarrowTopk = 16;      // chosen experts, at most (a lane each)

// v of the lane that the DPP control names, within the row of 16 lanes.
template <int CTRL>
__device__ __forceinline__ uint32_t row_move(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), CTRL, 0xF, 0xF, false));
}
template <int CTRL>
__device__ __forceinline__ float row_move(float v) {
  return __uint_as_float(row_move<CTRL>(__float_as_uint(v)));
}
template <int CTRL>
__device__ __forceinline__ double row_move(double v) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v));
  const uint64_t lo = row_move<CTRL>(static_cast<uint32_t>(b)), hi = row_move<CTRL>(static_cast<uint32_t>(b >> 32));
  return __longlong_as_double(static_cast<long long>(hi << 32 | lo));
}
// Lane distances 1 and 2, then the mirrors of 8 and of 16 lanes: after each
// step all lanes of 2, 4, 8 and 16 hold the same result.
constexpr int kSwap1 = 0xB1, kSwap2 = 0x4E, kMirror8 = 0x141, kMirror16 = 0x140;

__device__ __forceinline__ float row_sum(float v) {
  v += row_move<kSwap1>(v);
  v += row_move<kSwap2>(v);
  v += row_move<kMirror8>(v);
  return v + row_move<kMirror16>(v);
}
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, row_move<kSwap1>(v));
  v = fmaxf(v, row_move<kSwap2>(v));
  v = fmaxf(v, row_move<kMirror8>(v));
  return fmaxf(v, row_move<kMirror16>(v));
}

// e^x for x <= 0 (NaN and anything below -200: 0). x = (n + f) ln 2 with |f|
// at most a half, f exact to 2^-26 through a second term of 1 / ln 2, and 2^f
// by the instruction, good to one step; n goes into the exponent. 7
// instructions, without the library's branches for other x.
__device__ __forceinline__ float exp_below(float x) {
  constexpr float kHi = 1.4426950408889634f;
  constexpr float kLo = static_cast<float>(1.4426950408889634 - static_cast<double>(kHi));
  x = fmaxf(x, -200.0f);
  const float n = rintf(x * kHi);
  const float f = fmaf(x, kLo, fmaf(x, kHi, -n));
  return ldexpf(__builtin_amdgcn_exp2f(f), static_cast<int>(n));
}

// 1 / x for x >= 1: the instruction's one step of error, taken out by one
// Newton step (an infinite x gives 0).
__device__ __forceinline__ float reciprocal(float x) {
  const float r = __builtin_amdgcn_rcpf(x);
  return x < INFINITY ? fmaf(fmaf(-x, r, 1.0f), r, r) : 0.0f;
}

// A choice key with the expert's index in its low bits (the complement, so
// that of equal logits the lower index is larger): all keys differ, and one
// maximum finds both. 16-bit logits, seen as fp32, leave 13 low bits free, so
// their keys fit 32 bits; an fp32 logit's key and index go into the fraction
// of a double in [1, 2), whose maximum is one instruction too. kNone: masked.
template <typename T>
struct Key {
  using type = uint32_t;
  static constexpr uint32_t kField = 0x1fff;
  static __device__ __forceinline__ type none() { return 0; }
  static __device__ __forceinline__ type pack(float z, int i) {
    const uint32_t k = order_key(z);
    return k ? (k & ~kField) | (kField - static_cast<uint32_t>(i)) : 0;
  }
  static __device__ __forceinline__ int index(type k) { return k ? static_cast<int>(kField - (k & kField)) : -1; }
  static __device__ __forceinline__ float value(type k) {
    const uint32_t b = k >> 31 ? (k & ~kField) ^ 0x80000000u : ~(k | kField);
    return k ? __uint_as_float(b) : -INFINITY;
  }
};
template <>
struct Key<float> {
  using type = double;
  static constexpr uint32_t kField = 0x7ff;
  static __device__ __forceinline__ type none() { return 1.0; }
  static __device__ __forceinline__ type pack(float z, int i) {
    const uint32_t k = order_key(z);
    const uint64_t b = 0x3ff0000000000000ull | static_cast<uint64_t>(k) << 11 | (kField - static_cast<uint32_t>(i));
    return k ? __longlong_as_double(static_cast<long long>(b)) : none();
  }
  static __device__ __forceinline__ uint64_t bits(type k) {
    return static_cast<uint64_t>(__double_as_longlong(k)) & 0x000fffffffffffffull;
  }
  static __device__ __forceinline__ int index(type k) {
    const uint64_t b = bits(k);
    return b ? static_cast<int>(kField - (b & kField)) : -1;
  }
  static __device__ __forceinline__ float value(type k) {
    const uint32_t o = static_cast<uint32_t>(bits(k) >> 11);
    return o ? __uint_as_float(o >> 31 ? o ^ 0x80000000u : ~o) : -INFINITY;
  }
};

// A list that rises and falls once, sorted (largest first).
template <int N, typename K>
__device__ __forceinline__ void sort_merged(K (&a)[N]) {
#pragma unroll
  for (int d = N / 2; d > 0; d >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((i & d) == 0) {
        const K x = a[i], y = a[i + d];
        a[i] = larger(x, y);
        a[i + d] = smaller(x, y);
      }
}
template <int N, typename K>
__device__ __forceinline__ void sort_list(K (&a)[N]) {
#pragma unroll
  for (int k = 2; k <= N; k <<= 1)
#pragma unroll
    for (int d = k / 2; d > 0; d >>= 1)
#pragma unroll
      for (int i = 0; i < N; ++i)
        if ((i & d) == 0) {
          const K x = a[i], y = a[i + d];
          const bool falls = (i & k) == 0;
          a[i] = falls ? larger(x, y) : smaller(x, y);
          a[i + d] = falls ? smaller(x, y) : larger(x, y);
        }
}
// The N largest of two sorted lists, sorted.
template <int N, typename K>
__device__ __forceinline__ void merge_lists(K (&a)[N], const K (&b)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = larger(a[i], b[N - 1 - i]);
  sort_merged<N>(a);
}
template <int CTRL, int N, typename K>
__device__ __forceinline__ void merge_lanes(K (&a)[N]) {
  K b[N];
#pragma unroll
  for (int i = 0; i < N; ++i) b[i] = row_move<CTRL>(a[i]);
  merge_lists<N>(a, b);
}

// The row's N largest keys, sorted, in every lane of the row.
template <typename T, int VPL, int N>
__device__ __forceinline__ void row_best(const float (&z)[VPL], typename Key<T>::type (&best)[N]) {
  using K = typename Key<T>::type;
  const int i0 = static_cast<int>(threadIdx.x & (kRowLanes - 1)) * VPL;
#pragma unroll
  for (int at = 0; at < VPL; at += N) {
    K part[N];
#pragma unroll
    for (int i = 0; i < N; ++i) part[i] = at + i < VPL ? Key<T>::pack(z[at + i < VPL ? at + i : 0], i0 + at + i) : Key<T>::none();
    sort_list<N>(part);
    if (at == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) best[i] = part[i];
    } else {
      merge_lists<N>(best, part);
    }
  }
  merge_lanes<kSwap1, N>(best);
  merge_lanes<kSwap2, N>(best);
  merge_lanes<kMirror8, N>(best);
  merge_lanes<kMirror16, N>(best);
}

// A row's terms t_i (see row_terms) and their sum, by its 16 lanes.
template <int VPL, bool SIGMOID>
__device__ __forceinline__ float narrow_terms(const float (&z)[VPL], float (&t)[VPL]) {
  float m = z[0];
#pragma unroll
  for (int i = 1; i < VPL; ++i) m = fmaxf(m, z[i]);
  m = row_max(m);
  if constexpr (SIGMOID) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const float e = exp_below(-fabsf(z[i]));
      t[i] = (z[i] > 0.0f ? 1.0f : e) * reciprocal(1.0f + e);
    }
    if (__any(m < 0.0f)) {  // all logits of a row below 0: by the largest
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (m < 0.0f) t[i] = z[i] > -INFINITY ? exp_below(z[i] - m) * reciprocal(1.0f + exp_below(z[i])) : 0.0f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i) t[i] = exp_below(z[i] - m);
    if (__any(m == INFINITY)) {
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (m == INFINITY) t[i] = z[i] == m ? 1.0f : 0.0f;
    }
  }
  float s[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) s[i] = t[i];
#pragma unroll
  for (int d = VPL / 2; d > 0; d >>= 1)
#pragma unroll
    for (int i = 0; i < d; ++i) s[i] += s[i + d];
  return row_sum(s[0]);
}

// The weight of the row's k-th choice in its lane k, from the lane's own
// chosen logit (id -1: none), the row's largest logit and the sum of its terms
// (softmax over all experts only).
template <bool SIGMOID>
__device__ __forceinline__ float choice_weight(const Pick& pk, int id, float zc, float top, float all) {
  if constexpr (SIGMOID) {
    // In 64 bits; renormalised by the largest where all logits are below 0.
    const double shift = pk.renorm ? fminf(top, 0.0f) : 0.0, zd = zc;
    const double s = id < 0 ? 0.0 : zc > 0.0f ? 1.0 / (1.0 + exp(-zd)) : exp(zd - shift) / (1.0 + exp(zd));
    double sum = 1.0;
    if (pk.renorm) {
      sum = s;
      sum += row_move<kSwap1>(sum);
      sum += row_move<kSwap2>(sum);
      sum += row_move<kMirror8>(sum);
      sum += row_move<kMirror16>(sum);
    }
    return id < 0 ? 0.0f : static_cast<float>(s / sum * static_cast<double>(pk.scale));
  } else {
    const float e = id < 0 ? 0.0f : expf(below(zc, top));
    if (pk.renorm) all = row_sum(e);
    return id < 0 ? 0.0f : e / all * pk.scale;
  }
}

// The choice of a row from its N best: lane k's id and logit.
template <typename T, int N>
__device__ __forceinline__ void own_choice(const typename Key<T>::type (&best)[N], int topk, int& id, float& zc) {
  const int l = threadIdx.x & (kRowLanes - 1);
  typename Key<T>::type mine = Key<T>::none();
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i == l && i < topk) mine = best[i];
  id = Key<T>::index(mine);
  zc = Key<T>::value(mine);
}

template <typename T, int VPL, bool SIGMOID, int N>
__global__ void __launch_bounds__(kThreads) choose_narrow_kernel(Rows r, Pick pk, float* __restrict__ weights,
                                                                 int32_t* __restrict__ ids) {
  const int l = threadIdx.x & (kRowLanes - 1);
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kBlockRows + (threadIdx.x >> 4);
  const int64_t tc = t < r.T ? t : r.T - 1;
  const bool on = t < r.T && (!r.mask || r.mask[tc]);
  float z[VPL];
  load_part<T, VPL, kRowLanes>(static_cast<const T*>(r.logits) + tc * r.stride, r.E, r.vec, z);
  typename Key<T>::type best[N];
  row_best<T, VPL, N>(z, best);
  int id;
  float zc, all = 1.0f;
  own_choice<T, N>(best, pk.topk, id, zc);
  if constexpr (!SIGMOID) {
    if (!pk.renorm) {
      float term[VPL];
      all = narrow_terms<VPL, false>(z, term);
    }
  }
  const float w = choice_weight<SIGMOID>(pk, id, zc, Key<T>::value(best[0]), all);
  if (l < pk.topk && t < r.T) {
    ids[t * pk.topk + l] = on ? id : -1;
    weights[t * pk.topk + l] = on ? w : 0.0f;
  }
}

// balance_kernel with rows of 16 lanes: a workgroup takes kBlockRows rows of
// its sequence at a time, the next ones requested before the present ones are
// worked on. N 0: the choice is given.
template <typename T, int VPL, bool SIGMOID, int N>
__global__ void __launch_bounds__(kThreads) balance_narrow_kernel(Rows r, Pick pk, const void* __restrict__ given,
                                                                  int eb, float* __restrict__ weights,
                                                                  int32_t* __restrict__ ids, Partial out) {
  constexpr bool CHOOSE = N > 0;
  __shared__ int32_t s_count[kRowLanes * VPL];
  __shared__ float s_sum[kWaves][kRowLanes * VPL];
  __shared__ int s_valid[kWaves];
  const int tid = threadIdx.x, wave = tid >> 6, l = tid & (kRowLanes - 1);
  const int s = blockIdx.y, j = blockIdx.x, E = r.E;
  if (s == 0 && j == 0 && tid == 0) *out.done = 0;
  if (s == r.num_seqs) {
    if constexpr (CHOOSE) mark_padding(r, pk.topk, weights, ids, j, out.parts);
    return;
  }
  for (int i = tid; i < E; i += kThreads) s_count[i] = 0;
  __syncthreads();
  int64_t lo, hi;
  seq_range(r, s, lo, hi);
  const int64_t step = static_cast<int64_t>(out.parts) * kBlockRows;
  const T* const base = static_cast<const T*>(r.logits);
  float sum[VPL], next[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) sum[i] = 0.0f;
  int valid = 0;
  const int64_t t0 = lo + static_cast<int64_t>(j) * kBlockRows;
  auto clamped = [&](int64_t t) { return t < hi ? t : hi - 1; };
  if (t0 < hi) load_part<T, VPL, kRowLanes>(base + clamped(t0 + (tid >> 4)) * r.stride, E, r.vec, next);
  for (int64_t tb = t0; tb < hi; tb += step) {
    const int64_t t = tb + (tid >> 4);
    float z[VPL], term[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) z[i] = next[i];
    if (tb + step < hi) load_part<T, VPL, kRowLanes>(base + clamped(t + step) * r.stride, E, r.vec, next);
    const bool on = t < hi && (!r.mask || r.mask[t]);
    int64_t id = -1;
    if constexpr (!CHOOSE) {
      if (l < pk.topk && on) id = load_id(given, eb, t * pk.topk + l);
    }
    const float all = narrow_terms<VPL, SIGMOID>(z, term);
    if constexpr (CHOOSE) {
      typename Key<T>::type best[N];
      row_best<T, VPL, N>(z, best);
      int own;
      float zc;
      own_choice<T, N>(best, pk.topk, own, zc);
      const float w = choice_weight<SIGMOID>(pk, own, zc, Key<T>::value(best[0]), all);
      if (l < pk.topk && t < hi) {
        ids[t * pk.topk + l] = on ? own : -1;
        weights[t * pk.topk + l] = on ? w : 0.0f;
      }
      id = on ? own : -1;
    }
    if (id >= 0 && id < E) atomicAdd(&s_count[id], 1);
    const float inv = on && all > 0.0f ? 1.0f / all : 0.0f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) sum[i] = fmaf(term[i], inv, sum[i]);
    valid += on;
  }
  // The wave's four rows of lanes, then the waves.
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(sum[i]), __float_as_uint(sum[i]), false, false);
    const float v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    sum[i] = __uint_as_float(b[0]) + __uint_as_float(b[1]);
  }
  valid += __shfl_xor(valid, 16, 64);
  valid += __shfl_xor(valid, 32, 64);
  if ((tid & 63) < kRowLanes) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) s_sum[wave][l * VPL + i] = sum[i];
  }
  if ((tid & 63) == 0) s_valid[wave] = valid;
  __syncthreads();
  store_partial(out, s, j, E, s_count, &s_sum[0][0], kRowLanes * VPL, s_valid);
}

// The sequence of row t (the last that starts at or before it), and whether
// the row lies in it.
__device__ __forceinline__ bool find_seq(const Rows& r, int64_t t, int& s) {
  s = 0;
  if (!r.offsets) return true;
  int a = 0, z = r.num_seqs;
  while (z - a > 1) {
    const int m = (a + z) >> 1;
    if (r.offsets[m] <= t)
      a = m;
    else
      z = m;
  }
  s = a;
  return r.offsets[s] <= t && t < r.offsets[s + 1];
}

struct Back {
  const void* ids;
  int eb;
  const float* grad_weights;  // null: none
  const int32_t* counts;      // null: no loss
  const int32_t* tokens;
  const float* grad_loss;
  bool count_vec;  // rows of counts start on 16 bytes
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
  int s;
  const bool on = find_seq(r, t, s) && (!r.mask || r.mask[t]);
  float z[VPL], p[VPL], dz[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) dz[i] = 0.0f;
  if (on) {
    const T* row = static_cast<const T*>(r.logits) + t * r.stride;
    load_part<T, VPL, 64>(row, E, r.vec, z);
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

template <typename T, int VPL>
__device__ __forceinline__ void store_part(T* __restrict__ row, int E, bool vec, const float (&v)[VPL]) {
  constexpr int kBytes = VPL * static_cast<int>(sizeof(T));
  const int i0 = static_cast<int>(threadIdx.x & (kRowLanes - 1)) * VPL;
  if (kBytes >= 4 && vec && i0 + VPL <= E) {
    T o[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) store_as(&o[i], v[i]);
    if constexpr (kBytes % 16 == 0) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i)
        reinterpret_cast<u32x4*>(row + i0)[i] = reinterpret_cast<const u32x4*>(o)[i];
    } else if constexpr (kBytes == 8) {
      *reinterpret_cast<uint2*>(row + i0) = *reinterpret_cast<const uint2*>(o);
    } else if constexpr (kBytes == 4) {
      *reinterpret_cast<uint32_t*>(row + i0) = *reinterpret_cast<const uint32_t*>(o);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (i0 + i < E) store_as(row + i0 + i, v[i]);
  }
}

// The counts of a lane's experts (0 past E).
template <int VPL>
__device__ __forceinline__ void load_counts(const int32_t* __restrict__ row, int E, bool vec, float (&v)[VPL]) {
  const int i0 = static_cast<int>(threadIdx.x & (kRowLanes - 1)) * VPL;
  if (VPL % 4 == 0 && vec && i0 + VPL <= E) {
    u32x4 c[VPL / 4 > 0 ? VPL / 4 : 1];
#pragma unroll
    for (int i = 0; i < VPL / 4; ++i) c[i] = reinterpret_cast<const u32x4*>(row + i0)[i];
#pragma unroll
    for (int i = 0; i < VPL; ++i) v[i] = static_cast<float>(static_cast<int32_t>(c[i / 4][i % 4]));
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i) v[i] = i0 + i < E ? static_cast<float>(row[i0 + i]) : 0.0f;
  }
}

// backward_kernel with rows of 16 lanes. The chosen experts' own terms are
// added by the lane that holds the choice, which writes that element again
// behind the row's store, instead of a search for it among the row's lanes.
template <typename T, int VPL, bool SIGMOID>
__global__ void __launch_bounds__(kThreads) backward_narrow_kernel(Rows r, Pick pk, Back b, T* __restrict__ grad,
                                                                   bool grad_vec) {
  __shared__ uint8_t s_place[kBlockRows][kNarrowExperts];  // the last place of an expert in the row's choice
  const int l = threadIdx.x & (kRowLanes - 1), E = r.E;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kBlockRows + (threadIdx.x >> 4);
  const int64_t tc = t < r.T ? t : r.T - 1;
  const T* row = static_cast<const T*>(r.logits) + tc * r.stride;
  float z[VPL], p[VPL];
  load_part<T, VPL, kRowLanes>(row, E, r.vec, z);
  int s;
  const bool on = find_seq(r, tc, s) && (!r.mask || r.mask[tc]);
  int id = -1;
  float g = 0.0f, zc = -INFINITY;
  if (b.grad_weights && l < pk.topk) {
    const int64_t e = load_id(b.ids, b.eb, tc * pk.topk + l);
    id = e >= 0 && e < E ? static_cast<int>(e) : -1;
    if (id >= 0) {
      g = b.grad_weights[tc * pk.topk + l] * pk.scale;
      zc = to_float(row[id]);
      zc = zc > -INFINITY ? zc : -INFINITY;
      s_place[threadIdx.x >> 4][id] = static_cast<uint8_t>(l);
    }
  }
  float k = 0.0f;  // G_i = k counts_i
  const int32_t* count = nullptr;
  if (b.counts) {
    const float n = static_cast<float>(b.tokens[s]);
    k = n > 0.0f ? *b.grad_loss * static_cast<float>(E) /
                       (n * n * static_cast<float>(pk.topk) * static_cast<float>(b.tokens[r.num_seqs]))
                 : 0.0f;
    count = b.counts + static_cast<int64_t>(s) * E;
  }
  const float all = narrow_terms<VPL, SIGMOID>(z, p);
  const float inv = all > 0.0f ? 1.0f / all : 0.0f;
  float G[VPL], dot = 0.0f;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    p[i] *= inv;
    G[i] = 0.0f;
  }
  if (count) {
    load_counts<VPL>(count, E, b.count_vec, G);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      G[i] *= k;
      dot = fmaf(G[i], p[i], dot);
    }
  }
  // The lane's own choice: its share of the weights, probability and slope.
  float w = 0.0f, pc = 0.0f, slope = 1.0f, own = 0.0f;
  const bool mine = id >= 0 && on;
  if (b.grad_weights) {
    const float top = row_max(zc);
    const float ez = SIGMOID ? exp_below(-fabsf(zc)) : 0.0f;
    float e = 0.0f;
    if constexpr (SIGMOID) {
      const float inv1 = reciprocal(1.0f + ez);
      slope = (zc > 0.0f ? ez : 1.0f) * inv1;
      e = (zc > 0.0f ? 1.0f : exp_below(zc - fminf(top, 0.0f))) * inv1;
      own = (zc > 0.0f ? 1.0f : ez) * inv1;  // the score itself
    } else {
      e = exp_below(below(zc, top));
    }
    if (id < 0) e = 0.0f;
    if (pk.renorm) {
      const float sum = row_sum(e);
      w = sum > 0.0f ? e / sum : 0.0f;
    }
    // p_c: the row's own p at the chosen expert, from the same logit.
    float m = z[0];
#pragma unroll
    for (int i = 1; i < VPL; ++i) m = fmaxf(m, z[i]);
    m = row_max(m);
    if constexpr (SIGMOID)
      pc = (m < 0.0f ? exp_below(zc - m) * reciprocal(1.0f + ez) : own) * inv;
    else
      pc = exp_below(below(zc, m)) * inv;
    if (id < 0) pc = 0.0f;
    if (!SIGMOID && !pk.renorm) dot = fmaf(g, pc, dot);
  }
  if (count || (!SIGMOID && !pk.renorm)) dot = row_sum(dot);
  float dz[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    dz[i] = on ? p[i] * (G[i] - dot) : 0.0f;
    if (SIGMOID && count) {  // 1 - s
      const float e = exp_below(-fabsf(z[i]));
      dz[i] *= (z[i] > 0.0f ? e : 1.0f) * reciprocal(1.0f + e);
    }
  }
  if (t < r.T) store_part<T, VPL>(grad + t * E, E, grad_vec, dz);
  if (b.grad_weights) {
    const float gw = pk.renorm ? row_sum(g * w) : 0.0f;
    float v = pc * ((count && id >= 0 ? k * static_cast<float>(count[id]) : 0.0f) - dot);
    if (SIGMOID) v *= slope;
    float term = pk.renorm ? w * slope * (g - gw) : SIGMOID ? g * own * slope : pc * g;
    // An expert that stands in the row several times (a given choice): each of
    // its places takes the sum of their terms, in the order of the places.
    // (The look costs 0.2 us of 13.3 to 13.9: 32768 tokens of 256 experts, top-8,
    // bf16.) The row's places were written by this wave.
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (__any(id >= 0 && s_place[threadIdx.x >> 4][id] != l)) {
      const float one = term;
      term = 0.0f;
      for (int i = 0; i < pk.topk; ++i) {
        const int other = __shfl(id, i, kRowLanes);
        const float theirs = __shfl(one, i, kRowLanes);
        if (other == id) term += theirs;
      }
    }
    v += term;
    // Behind the row's store, and kept there: the two go to the same address.
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    if (mine && t < r.T) store_as(grad + t * E + id, v);
  }
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
  XP_REQUIRE(scale >= -FLT_MAX && scale <= FLT_MAX, "%s: scale must be a finite fp32 value", what);
  return XP_OK;
}

size_t elem_bytes(int dtype) { return dtype == XP_FLOAT32 ? 4 : 2; }

// The experts a lane holds: the least power of two that covers E.
int values_per_lane(int64_t E, int lanes) {
  int v = 1;
  while (lanes * v < E) v *= 2;
  return v;
}

// Whether rows are 16 lanes' (see the top). us in a graph by that form and by a
// wave per row, 32768 tokens, choice alone | choice and loss | with the backward:
//   8 experts, top-2, bf16             5.0 and 9.7 | 12 and 28 | 17 and 42
//   256 experts, top-16, fp32          17 and 39 | 30 and 92 | 50 and 126
//   512 experts, top-10, bf16          20 and 35 | 37 and 91 | 63 and 145
//   512 experts, top-16, fp32          25 and 50 | 42 and 118 | 84 and 203
//   the same by the sigmoid            25 and 53 | 59 and 150 | 106 and 225
// At 64 tokens the choice alone is the slower one for some (64 experts, fp32, 3.2
// and 2.8; 384, whose lanes do not share them evenly, 6.0 and 5.0), with the loss
// none is (8.4 and 11.3; 13.2 and 22.6). Beyond the rule: 1024 experts, top-8, 44 |
// 111 | 249 for 32768 tokens; 256 experts, top-33, 70 | 157 | 203.
bool narrow_rows(int64_t E, int64_t topk) { return E <= kNarrowExperts && topk <= kNarrowTopk; }

Rows rows_of(const Call& c, int lanes) {
  const size_t eb = elem_bytes(c.dtype), chunk = std::min<size_t>(16, values_per_lane(c.E, lanes) * eb);
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

// Workgroups that share a sequence: kBlockRows rows each at least, and no more
// than about 512 in all (the join reads a row of E sums from each). Every
// sequence gets as many, by their average length: one that holds most of the
// rows is done by its own few, and its sums run over as many more rows each
// (choice and loss of 32768 tokens, 256 experts: 40 even sequences 37 us, one of
// 32000 rows among 40 344; 512 even ones 209, one of 32000 rows among 512 4020).
int balance_parts(int64_t T, int64_t num_seqs) {
  const int64_t per = (T + num_seqs - 1) / num_seqs;
  const int64_t parts = std::min<int64_t>((per + kBlockRows - 1) / kBlockRows, std::max<int64_t>(1, 512 / num_seqs));
  return static_cast<int>(std::max<int64_t>(parts, 1));
}

// The grid of a launch of `per_block` rows a workgroup: fewer than 2^32 threads.
int row_grid(const Call& c, int per_block, dim3* grid) {
  const int64_t blocks = (c.T + per_block - 1) / per_block;
  if (blocks * kThreads > UINT32_MAX)
    return fail(XP_E_LIMIT, "%s: %lld rows exceed the launch grid", c.what, (long long)c.T);
  *grid = dim3(static_cast<unsigned>(blocks));
  return XP_OK;
}

int64_t align256(int64_t n) { return (n + 255) & ~int64_t(255); }

int64_t join_blocks(int64_t E) { return (E + kJoinExperts - 1) / kJoinExperts; }

int64_t balance_layout(int64_t T, int64_t E, int64_t num_seqs, Partial* p, uint8_t* base) {
  const int64_t parts = balance_parts(T, num_seqs), n = parts * num_seqs;
  const int64_t sz[4] = {align256(n * E * 8), align256(n * 4), align256(num_seqs * join_blocks(E) * 8), 256};
  if (p) {
    p->parts = static_cast<int>(parts);
    p->pc = reinterpret_cast<uint2*>(base);
    p->n = reinterpret_cast<int32_t*>(base + sz[0]);
    p->loss = reinterpret_cast<double*>(base + sz[0] + sz[1]);
    p->done = reinterpret_cast<int32_t*>(base + sz[0] + sz[1] + sz[2]);
  }
  return sz[0] + sz[1] + sz[2] + sz[3];
}

int launch_balance(const Call& c, const Pick& pk, bool choose, const void* given, int eb, float* weights, int32_t* ids,
                   void* work, int32_t* counts, int32_t* tokens, float* loss, void* stream) {
  const hipStream_t st = as_stream(stream);
  Partial part{};
  balance_layout(c.T, c.E, c.num_seqs, &part, static_cast<uint8_t*>(work));
  const dim3 grid(static_cast<unsigned>(part.parts), static_cast<unsigned>(c.num_seqs + (choose && c.offsets ? 1 : 0)));
  const bool narrow = narrow_rows(c.E, pk.topk) && !pk.bias && pk.groups == 1;
  const int lanes = narrow ? kRowLanes : 64;
  const Rows r = rows_of(c, lanes);
  const bool wide = choose && pk.bias;
  const size_t keys = choose && pk.groups > 1 ? static_cast<size_t>(kWaves) * c.E * (wide ? 8 : 4) : 0;
  const size_t lds =
      narrow ? 0 : ((c.E * 4 + 15) & ~size_t(15)) + std::max(keys, static_cast<size_t>(kWaves) * c.E * 4);
  dispatch(c.dtype, values_per_lane(c.E, lanes), [&](auto type, auto v) {
    using T = decltype(type);
    constexpr int V = decltype(v)::value;
    auto go = [&](auto* kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(kThreads), lds, st, r, pk, given, eb, weights, ids, part);
    };
    auto by_score = [&](auto sig) {
      constexpr bool S = decltype(sig)::value != 0;
      if (narrow)
        !choose ? go(balance_narrow_kernel<T, V, S, 0>)
                : pk.topk <= 8 ? go(balance_narrow_kernel<T, V, S, 8>) : go(balance_narrow_kernel<T, V, S, 16>);
      else
        !choose ? go(balance_kernel<T, V, S, false, false>)
                : wide ? go(balance_kernel<T, V, S, true, true>) : go(balance_kernel<T, V, S, true, false>);
    };
    pk.sigmoid ? by_score(Int<1>{}) : by_score(Int<0>{});
  });
  if (int rc = check_launch("balance_kernel")) return rc;
  hipLaunchKernelGGL(balance_join_kernel,
                     dim3(static_cast<unsigned>(join_blocks(c.E)), static_cast<unsigned>(c.num_seqs)), dim3(kThreads), 0,
                     st, part, static_cast<int>(c.E), pk.topk, static_cast<int>(c.num_seqs), counts, tokens, loss);
  return check_launch("balance_join_kernel");
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
  const bool narrow = narrow_rows(E, topk) && !bias && groups == 1;
  const int lanes = narrow ? kRowLanes : 64, per_block = narrow ? kBlockRows : kWaves;
  const Rows r = rows_of(c, lanes);
  const size_t lds = groups > 1 ? static_cast<size_t>(kWaves) * E * (bias ? 8 : 4) : 0;
  dim3 grid;
  if (int rc = row_grid(c, per_block, &grid)) return rc;
  dispatch(dtype, values_per_lane(E, lanes), [&](auto type, auto v) {
    using L = decltype(type);
    constexpr int V = decltype(v)::value;
    auto go = [&](auto* kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(kThreads), lds, as_stream(stream), r, pk, weights, ids);
    };
    if (!narrow)
      bias ? go(choose_kernel<L, V, true>) : go(choose_kernel<L, V, false>);
    else if (topk <= 8)
      pk.sigmoid ? go(choose_narrow_kernel<L, V, true, 8>) : go(choose_narrow_kernel<L, V, false, 8>);
    else
      pk.sigmoid ? go(choose_narrow_kernel<L, V, true, 16>) : go(choose_narrow_kernel<L, V, false, 16>);
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
  XP_REQUIRE(scale >= -FLT_MAX && scale <= FLT_MAX, "%s: scale must be a finite fp32 value", what);
  if (T == 0) return XP_OK;
  XP_REQUIRE(grad, "%s: null gradient", what);
  const Pick pk{static_cast<int>(topk), scoring == XP_SCORE_SIGMOID, renormalize != 0, 1, 1, static_cast<float>(scale),
                nullptr};
  const Back b{topk_ids, topk_elem_bytes, grad_weights, counts, tokens, grad_loss, E % 4 == 0 && aligned16(counts)};
  const bool narrow = narrow_rows(E, topk);
  const int lanes = narrow ? kRowLanes : 64, per_block = narrow ? kBlockRows : kWaves;
  const Rows r = rows_of(c, lanes);
  dim3 grid;
  if (int rc = row_grid(c, per_block, &grid)) return rc;
  dispatch(dtype, values_per_lane(E, lanes), [&](auto type, auto v) {
    using L = decltype(type);
    constexpr int V = decltype(v)::value;
    const size_t chunk = std::min<size_t>(16, V * sizeof(L));
    const bool vec = reinterpret_cast<uintptr_t>(grad) % chunk == 0 && E * sizeof(L) % chunk == 0;
    if (narrow) {
      auto* kernel = pk.sigmoid ? backward_narrow_kernel<L, V, true> : backward_narrow_kernel<L, V, false>;
      hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, as_stream(stream), r, pk, b, static_cast<L*>(grad), vec);
    } else {
      auto* kernel = pk.sigmoid ? backward_kernel<L, V, true> : backward_kernel<L, V, false>;
      hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, as_stream(stream), r, pk, b, static_cast<L*>(grad));
    }
  });
  return check_launch("backward_kernel");
}

}  // extern "C"

// Low-rank adapters of many requests beside the experts' projections.
//
// Pair p = (token t, choice k) has the adapter of its token's request and the
// expert of its choice. Its row of a projection gets
//   scale B (A x)        A: [R][K], B: [n][R] of that (adapter, expert)
// per slice (gate and up are two slices with matrices of their own).
//
// The pairs of one (adapter, expert), a group, are multiplied together, 16 at
// a time (a tile): u = A x over K, split over the workgroup's waves and summed
// in LDS, then B u over the workgroup's columns, with the 16x16x32 matrix
// instruction, the matrices as its first operand, so that a lane's four
// outputs are four consecutive columns of one pair. Both products are one
// launch: a workgroup has its tile's u whole, and nothing but the result goes
// to memory. Bound by the bytes of A and B: with the top-k of hundreds of
// experts a group has few pairs.
//
// u enters the second product as the sum of two values of the operands' type,
// its rounding and the rounding of what is left, so no more than 2^-16 of it
// is lost (one rounding to bf16 would lose 2^-9). fp16 covers 2^-14 to 2^16
// with full precision, so there a pair's u is first scaled by a power of two
// that puts its largest value near 2^13, and the result scaled back.
//
// Grouping. Up to 64 pairs every wave groups them itself, a pair per lane.
// Above, one launch of up to 256 workgroups, each of which owns a range of
// groups: it reads every pair's group, counts those of its range and those
// below it, and writes its part of the list. A tile's place needs no count of
// the tiles before it: a range with pb pairs and gb groups below it starts at
// pb / 16 + min(gb, pb), which leaves room for its tiles whatever their
// sizes; unused places are marked empty.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <type_traits>

#include "common.h"

namespace xp {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kTile = 16;             // pairs per tile
constexpr int kDirectPairs = 64;      // pairs that a wave groups itself
constexpr int kGroupThreads = 1024;
constexpr int kRangeGroups = 4096;    // groups a grouping workgroup counts in LDS, at most
constexpr int64_t kMaxGroups = (1 << 20) - 1;

struct Bf16 {
  static __device__ __forceinline__ uint16_t bits(float v) {
    __hip_bfloat16 b = __float2bfloat16(v);
    return *reinterpret_cast<uint16_t*>(&b);
  }
  static __device__ __forceinline__ float value(uint16_t b) { return __uint_as_float(static_cast<uint32_t>(b) << 16); }
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  }
  static constexpr bool kScaled = false;
};
struct Fp16 {
  static __device__ __forceinline__ uint16_t bits(float v) {
    __half h = __float2half(v);
    return *reinterpret_cast<uint16_t*>(&h);
  }
  static __device__ __forceinline__ float value(uint16_t b) {
    __half h = *reinterpret_cast<__half*>(&b);
    return __half2float(h);
  }
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  }
  static constexpr bool kScaled = true;
};

struct Ids {
  const void* adapter;
  const void* expert;  // null: expert 0
  int aeb, eeb;
  const int32_t* expert_map;  // null: every pair is listed
  int slots;
  int topk, adapters, experts;
};

// Pair p's group: adapter * experts + expert, adapters * experts for a pair
// without an adapter, -1 for one that is not listed.
__device__ __forceinline__ int pair_group(const Ids& d, int64_t p) {
  const int64_t e = d.expert ? load_id(d.expert, d.eeb, p) : 0;
  const int64_t a = load_id(d.adapter, d.aeb, static_cast<uint32_t>(p) / static_cast<uint32_t>(d.topk));
  const bool known = e >= 0 && e < d.experts;
  if (d.expert_map) {
    const int s = known ? d.expert_map[e] : -1;
    if (s < 0 || s >= d.slots) return -1;
  }
  return known && a >= 0 && a < d.adapters ? static_cast<int>(a * d.experts + e) : d.adapters * d.experts;
}

struct Entry {
  int group, first, count;  // count 0: no tile
  int pad;
};

// Exclusive scan of two counters over the workgroup of kGroupThreads.
__device__ __forceinline__ int2 block_scan2(int2 v, int2* s_tot) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int2 in = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int a = __shfl_up(in.x, off, 64), b = __shfl_up(in.y, off, 64);
    if (lane >= off) {
      in.x += a;
      in.y += b;
    }
  }
  if (lane == 63) s_tot[wave] = in;
  __syncthreads();
  int2 base = make_int2(0, 0);
  for (int w = 0; w < kGroupThreads / 64; ++w) {
    const int2 t = s_tot[w];
    if (w < wave) {
      base.x += t.x;
      base.y += t.y;
    }
  }
  return make_int2(base.x + in.x - v.x, base.y + in.y - v.y);
}

// Workgroup w lists the groups [w per, (w + 1) per): pairs[] by group, and a
// tile entry per kTile pairs of a group.
__global__ void __launch_bounds__(kGroupThreads) group_kernel(Ids d, int64_t npairs, int per,
                                                              int32_t* __restrict__ pairs,
                                                              Entry* __restrict__ tiles) {
  constexpr int kEach = kRangeGroups / kGroupThreads;
  __shared__ int s_count[kRangeGroups];
  __shared__ int2 s_tot[kGroupThreads / 64];
  __shared__ int s_below, s_own;
  const int tid = threadIdx.x;
  const int groups = d.adapters * d.experts + 1;
  const int g0 = blockIdx.x * per, g1 = g0 + per < groups ? g0 + per : groups;
  for (int i = tid; i < per; i += kGroupThreads) s_count[i] = 0;
  if (tid == 0) s_below = s_own = 0;
  __syncthreads();
  int below = 0, own = 0;
  for (int64_t p = tid; p < npairs; p += kGroupThreads) {
    const int g = pair_group(d, p);
    if (g < 0) continue;
    if (g < g0) {
      ++below;
    } else if (g < g1) {
      ++own;
      atomicAdd(&s_count[g - g0], 1);
    }
  }
  atomicAdd(&s_below, below);
  atomicAdd(&s_own, own);
  __syncthreads();
  const int pb = s_below, all = s_own;
  // A thread's kEach consecutive groups: first pair and first tile.
  int c[kEach];
  int2 mine = make_int2(0, 0);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int g = tid * kEach + i;
    c[i] = g < g1 - g0 ? s_count[g] : 0;
    mine.x += c[i];
    mine.y += (c[i] + kTile - 1) / kTile;
  }
  int2 at = block_scan2(mine, s_tot);  // (a barrier: the counts are read)
  const int below_groups = g0 < groups ? g0 : groups;
  const int own_groups = g1 > g0 ? g1 - g0 : 0;
  const int first = pb / kTile + (below_groups < pb ? below_groups : pb);
  const int upto = below_groups + own_groups, pe = pb + all;
  const int last = pe / kTile + (upto < pe ? upto : pe);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int g = tid * kEach + i;
    if (g < g1 - g0) s_count[g] = pb + at.x;  // where the group's next pair goes
    for (int k = 0; k < c[i]; k += kTile)
      tiles[first + at.y++] = Entry{g0 + g, pb + at.x + k, c[i] - k < kTile ? c[i] - k : kTile, 0};
    at.x += c[i];
  }
  __syncthreads();
  int used = 0;
  for (int w = 0; w < kGroupThreads / 64; ++w) used += s_tot[w].y;
  for (int i = first + used + tid; i < last; i += kGroupThreads) tiles[i] = Entry{0, 0, 0, 0};
  // The places behind the last range, by the last workgroup.
  if (blockIdx.x == gridDim.x - 1) {
    const int64_t bound = npairs / kTile + (groups < npairs ? groups : npairs);
    for (int64_t i = last + tid; i < bound; i += kGroupThreads) tiles[i] = Entry{0, 0, 0, 0};
  }
  for (int64_t p = tid; p < npairs; p += kGroupThreads) {
    const int g = pair_group(d, p);
    if (g >= g0 && g < g1) pairs[atomicAdd(&s_count[g - g0], 1)] = static_cast<int32_t>(p);
  }
}

struct Apply {
  const uint16_t* x;
  int64_t x_stride;
  int per_pair;
  int64_t K, Kp;
  const uint16_t* a;
  const uint16_t* b;
  const float* scales;
  const int32_t* ranks;
  int slices, n, np;
  const uint16_t* base;
  int64_t base_stride;
  uint16_t* out;
  int64_t out_stride;
  int64_t npairs;
  int nsplit;    // column parts per slice
  int tiles;     // places of the tile list
};

__device__ __forceinline__ float row16_max(float v) {
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xB1, 0xF, 0xF, false)));
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4E, 0xF, 0xF, false)));
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x141, 0xF, 0xF, false)));
  return fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x140, 0xF, 0xF, false)));
}

// Tile i of up to 64 pairs that are grouped here, by one wave (each does it
// for itself): the group, and row r's pair in lane r (0 .. 15).
__device__ __forceinline__ bool direct_tile(const Ids& d, int npairs, int i, int& group, int& count, int& row_pair) {
  const int lane = threadIdx.x & 63;
  const int g = lane < npairs ? pair_group(d, lane) : -1;
  unsigned long long same = __ballot(g >= 0);
  const int bits = 32 - __clz(d.adapters * d.experts);
  for (int b = 0; b < bits; ++b) {
    const bool set = (g >> b) & 1;
    const unsigned long long m = __ballot(set);
    same &= set ? m : ~m;
  }
  const int rank = static_cast<int>(lane_prefix(same));
  const int ntile = g >= 0 && rank == 0 ? (__popcll(same) + kTile - 1) / kTile : 0;
  int start = 0;
#pragma unroll
  for (int b = 0; b < 3; ++b) start += static_cast<int>(lane_prefix(__ballot((ntile >> b) & 1))) << b;
  const unsigned long long own = __ballot(ntile > 0 && start <= i && i < start + ntile);
  if (own == 0) return false;
  const int lead = __ffsll(static_cast<long long>(own)) - 1;
  group = __builtin_amdgcn_readlane(g, lead);
  const int r0 = (i - __builtin_amdgcn_readlane(start, lead)) * kTile;
  const int all = __popcll(__ballot(g == group));
  count = all - r0 < kTile ? all - r0 : kTile;
  const int r = rank - r0;
  const bool in = g == group && r >= 0 && r < kTile;
  // Row r's pair goes to lane r; the other lanes' go to lane 63.
  row_pair = __builtin_amdgcn_ds_permute(4 * (in ? r : 63), lane);
  return true;
}

// RB: 16-row blocks of a slice's rank. SPW: slices per workgroup.
template <typename T, int RB, int SPW>
__global__ void __launch_bounds__(kThreads) lora_kernel(Ids d, Apply p, const int32_t* __restrict__ pairs,
                                                        const Entry* __restrict__ tiles) {
  constexpr int NB = RB * SPW, R = 16 * RB;
  constexpr int kRow = R + 8;  // an LDS row of u: 16 bytes more, so that the rows spread over the banks
  __shared__ int s_pair[kTile];
  __shared__ __attribute__((aligned(16))) float s_u[kWaves][NB][16][kTile + 1];
  __shared__ __attribute__((aligned(16))) uint16_t s_hi[SPW][kTile][kRow], s_lo[SPW][kTile][kRow];
  __shared__ float s_back[SPW][kTile];

  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int q = lane >> 4, j = lane & 15;
  // Every XCD takes a contiguous part of the tile list, a tile's parts side
  // by side, so that the tiles of a group read its matrices into one L2.
  const int parts = p.slices / SPW * p.nsplit;
  const int per_xcd = (p.tiles + 7) / 8;
  const int xcd = blockIdx.x & 7, at = blockIdx.x >> 3;
  const int ti = xcd * per_xcd + at / parts, part = at % parts;
  if (at / parts >= per_xcd || ti >= p.tiles) return;
  const int s0 = part / p.nsplit * SPW, split = part % p.nsplit;

  int group, count;
  if (pairs) {
    const Entry e = tiles[ti];
    if (e.count == 0) return;
    group = e.group;
    count = e.count;
    if (tid < kTile) s_pair[tid] = pairs[e.first + (tid < count ? tid : 0)];
  } else {
    int row_pair;
    if (!direct_tile(d, static_cast<int>(p.npairs), ti, group, count, row_pair)) return;
    const int first = __builtin_amdgcn_readlane(row_pair, 0);
    if (tid < kTile) s_pair[tid] = tid < count ? row_pair : first;
  }
  __syncthreads();

  // This workgroup's 16-column blocks of a slice.
  const int blocks = p.np / 16, per_split = (blocks + p.nsplit - 1) / p.nsplit;
  const int b0 = split * per_split, b1 = b0 + per_split < blocks ? b0 + per_split : blocks;

  if (group == d.adapters * d.experts) {  // no adapter: base, or zeros
    if (p.out == p.base) return;
    const int c0 = b0 * 2, c1 = (b1 * 16 < p.n ? b1 * 16 : p.n) / 8;  // 8-column pieces
    for (int s = s0; s < s0 + SPW; ++s)
      for (int i = tid; i < count * (c1 - c0); i += kThreads) {
        const int r = i / (c1 - c0), c = s * p.n + (c0 + i - r * (c1 - c0)) * 8;
        const int64_t pr = s_pair[r];
        u32x4 v = {0, 0, 0, 0};
        if (p.base) v = *reinterpret_cast<const u32x4*>(p.base + pr * p.base_stride + c);
        *reinterpret_cast<u32x4*>(p.out + pr * p.out_stride + c) = v;
      }
    return;
  }
  const int adapter = group / d.experts;
  int rank = p.ranks[adapter];
  rank = rank < 0 ? 0 : (rank < R ? rank : R);

  // u = A x: wave w takes the K steps w, w + 4, ...
  const int my_pair = s_pair[j];
  const uint16_t* xrow = p.x + (p.per_pair ? my_pair : my_pair / d.topk) * p.x_stride;
  const uint16_t* arow = p.a + ((static_cast<int64_t>(group) * p.slices + s0) * R + j) * p.Kp + 8 * q;
  const int live = (rank + 15) / 16;  // blocks of a slice that hold anything
  f32x4 acc[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int steps = static_cast<int>(p.Kp / 32);
  for (int k = wave; k < steps; k += kWaves) {
    u32x4 xv = {0, 0, 0, 0};
    if (32 * k + 8 * q < p.K) xv = *reinterpret_cast<const u32x4*>(xrow + 32 * k + 8 * q);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      if (i % RB >= live) continue;
      const u32x4 av = *reinterpret_cast<const u32x4*>(arow + static_cast<int64_t>(16 * i) * p.Kp + 32 * k);
      acc[i] = T::mfma(av, xv, acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) s_u[wave][i][4 * q + r][j] = acc[i][r];
  __syncthreads();
  // The waves' sums, and u in two values: 16 threads per pair.
  {
    const int pr = tid >> 4, t16 = tid & 15;
#pragma unroll
    for (int s = 0; s < SPW; ++s) {
      float u[RB];
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        float v = s_u[0][s * RB + i][t16][pr];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) v += s_u[w][s * RB + i][t16][pr];
        u[i] = 16 * i + t16 < rank ? v : 0.0f;  // zero columns of A times an infinite x are not zero
        if (fabsf(u[i]) < INFINITY) top = fmaxf(top, fabsf(u[i]));
      }
      float up = 1.0f, back = 1.0f;
      if constexpr (T::kScaled) {
        top = row16_max(top);
        int e = 14;
        if (top > 0.0f) frexpf(top, &e);
        e = e < -110 ? -110 : e;
        up = ldexpf(1.0f, 14 - e);
        back = ldexpf(1.0f, e - 14);
      }
      if (t16 == 0) s_back[s][pr] = back;
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const float v = u[i] * up;
        const uint16_t hi = T::bits(v);
        const float rest = v - T::value(hi);
        s_hi[s][pr][16 * i + t16] = hi;
        s_lo[s][pr][16 * i + t16] = fabsf(T::value(hi)) < INFINITY ? T::bits(rest) : 0;
      }
    }
  }
  __syncthreads();

  // B u for this workgroup's columns.
  const float scale = p.scales[adapter];
  const int64_t pr = my_pair;
#pragma unroll
  for (int s = 0; s < SPW; ++s) {
    const uint16_t* bmat = p.b + (static_cast<int64_t>(group) * p.slices + s0 + s) * p.np * R;
    const float f = scale * s_back[s][j];
    // RB = 1: the lanes of the upper half of the instruction's 32 take what
    // is left of u, with the same 16 columns of B.
    constexpr int KS = RB == 1 ? 1 : RB / 2;
    u32x4 hi[KS], lo[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      if constexpr (RB == 1) {
        hi[0] = *reinterpret_cast<const u32x4*>(q < 2 ? &s_hi[s][j][8 * q] : &s_lo[s][j][8 * (q - 2)]);
      } else {
        hi[k] = *reinterpret_cast<const u32x4*>(&s_hi[s][j][32 * k + 8 * q]);
        lo[k] = *reinterpret_cast<const u32x4*>(&s_lo[s][j][32 * k + 8 * q]);
      }
    }
    for (int blk = b0 + wave; blk < b1; blk += kWaves) {
      const uint16_t* brow = bmat + static_cast<int64_t>(16 * blk + j) * R + 8 * (RB == 1 ? q & 1 : q);
      f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        if (32 * k >= rank) continue;
        const u32x4 bv = *reinterpret_cast<const u32x4*>(brow + 32 * k);
        y = T::mfma(bv, hi[k], y);
        if constexpr (RB > 1) y = T::mfma(bv, lo[k], y);
      }
      const int c = 16 * blk + 4 * q;
      if (j < count && c < p.n) {
        const int64_t col = static_cast<int64_t>(s0 + s) * p.n + c;
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = y[r] * f;
        if (p.base) {
          const u32x2 w = *reinterpret_cast<const u32x2*>(p.base + pr * p.base_stride + col);
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] += T::value(static_cast<uint16_t>(w[r >> 1] >> (16 * (r & 1))));
        }
        u32x2 o;
        o[0] = T::bits(v[0]) | static_cast<uint32_t>(T::bits(v[1])) << 16;
        o[1] = T::bits(v[2]) | static_cast<uint32_t>(T::bits(v[3])) << 16;
        *reinterpret_cast<u32x2*>(p.out + pr * p.out_stride + col) = o;
      }
    }
  }
}

// ---- host side ----

int64_t align256(int64_t n) { return (n + 255) & ~int64_t(255); }

// Places of the tile list: npairs / 16 + min(groups, npairs), the group of the pairs without an adapter among them.
int64_t tile_places(int64_t npairs, int64_t adapters, int64_t experts) {
  return npairs / kTile + std::min(adapters * experts + 1, npairs);
}

struct Listing {
  int32_t* pairs;
  Entry* tiles;
};

int64_t listing_layout(int64_t npairs, int64_t adapters, int64_t experts, Listing* w, uint8_t* base) {
  const int64_t sz = align256(npairs * 4);
  if (w) {
    w->pairs = reinterpret_cast<int32_t*>(base);
    w->tiles = reinterpret_cast<Entry*>(base + sz);
  }
  return sz + align256(tile_places(npairs, adapters, experts) * static_cast<int64_t>(sizeof(Entry)));
}

int check_ids(const char* what, const void* adapter_ids, int aeb, const void* topk_ids, int eb, int64_t T, int64_t topk,
              const int32_t* expert_map, int64_t slots, int64_t adapters, int64_t experts, Ids* d) {
  XP_REQUIRE(T >= 0 && topk >= 1 && topk <= INT32_MAX && T <= INT32_MAX && T * topk <= INT32_MAX,
             "%s: T=%lld, topk=%lld", what, (long long)T, (long long)topk);
  XP_REQUIRE(adapters >= 1 && experts >= 1 && adapters <= kMaxGroups && experts <= kMaxGroups &&
                 adapters * experts <= kMaxGroups,
             "%s: %lld adapters of %lld experts (at most %lld together)", what, (long long)adapters, (long long)experts,
             (long long)kMaxGroups);
  XP_REQUIRE((aeb == 4 || aeb == 8) && (eb == 4 || eb == 8), "%s: id sizes %d and %d", what, aeb, eb);
  XP_REQUIRE(topk_ids || experts == 1, "%s: %lld experts need topk_ids", what, (long long)experts);
  XP_REQUIRE(expert_map == nullptr || (slots >= 0 && slots <= INT32_MAX), "%s: %lld slots", what, (long long)slots);
  XP_REQUIRE(T == 0 || adapter_ids, "%s: null adapter ids", what);
  *d = Ids{adapter_ids, topk_ids, aeb, eb, expert_map, static_cast<int>(slots), static_cast<int>(topk),
           static_cast<int>(adapters), static_cast<int>(experts)};
  return XP_OK;
}

int check_listing(const char* what, int64_t npairs, int64_t adapters, int64_t experts, const void* work, int64_t bytes) {
  const int64_t need = listing_layout(npairs, adapters, experts, nullptr, nullptr);
  XP_REQUIRE(work && (reinterpret_cast<uintptr_t>(work) & 255) == 0 && bytes >= need,
             "%s: the workspace must be 256-byte aligned and of %lld B", what, (long long)need);
  return XP_OK;
}

int launch_group(const Ids& d, int64_t npairs, void* work, void* stream) {
  Listing w;
  listing_layout(npairs, d.adapters, d.experts, &w, static_cast<uint8_t*>(work));
  const int64_t groups = static_cast<int64_t>(d.adapters) * d.experts + 1;
  // More pairs take longer to scatter than to read: more workgroups, each with a part of the groups.
  int64_t wg = std::min<int64_t>(groups, npairs > 2048 ? 64 : 16);
  wg = std::max(wg, (groups + kRangeGroups - 1) / kRangeGroups);
  const int64_t per = (groups + wg - 1) / wg;
  hipLaunchKernelGGL(group_kernel, dim3(static_cast<unsigned>((groups + per - 1) / per)), dim3(kGroupThreads), 0,
                     as_stream(stream), d, npairs, static_cast<int>(per), w.pairs, w.tiles);
  return check_launch("group_kernel");
}

}  // namespace
}  // namespace xp

using namespace xp;

extern "C" {

int64_t xp_lora_workspace_bytes(int64_t npairs, int64_t adapters, int64_t experts) {
  if (npairs <= 0 || adapters <= 0 || experts <= 0 || adapters > kMaxGroups || experts > kMaxGroups) return 0;
  return listing_layout(npairs, adapters, experts, nullptr, nullptr);
}

int xp_lora_group(const void* adapter_ids, int adapter_elem_bytes, const void* topk_ids, int topk_elem_bytes, int64_t T,
                  int64_t topk, const int32_t* expert_map, int64_t slots, int64_t adapters, int64_t experts, void* work,
                  int64_t work_bytes, void* stream) {
  Ids d;
  if (int rc = check_ids("xp_lora_group", adapter_ids, adapter_elem_bytes, topk_ids, topk_elem_bytes, T, topk,
                         expert_map, slots, adapters, experts, &d))
    return rc;
  if (T == 0) return XP_OK;
  if (int rc = check_listing("xp_lora_group", T * topk, adapters, experts, work, work_bytes)) return rc;
  return launch_group(d, T * topk, work, stream);
}

int xp_lora_apply(const void* x, int dtype, int64_t x_stride, int per_pair, int64_t T, int64_t topk, int64_t K,
                  const void* a, const void* b, const float* scales, const int32_t* ranks, int64_t adapters,
                  int64_t experts, int64_t slices, int64_t n, int64_t R, const void* adapter_ids,
                  int adapter_elem_bytes, const void* topk_ids, int topk_elem_bytes, const int32_t* expert_map,
                  int64_t slots, const void* base, int64_t base_stride, void* out, int64_t out_stride, void* work,
                  int64_t work_bytes, int grouped, void* stream) {
  const char* what = "xp_lora_apply";
  Ids d;
  if (int rc = check_ids(what, adapter_ids, adapter_elem_bytes, topk_ids, topk_elem_bytes, T, topk, expert_map, slots,
                         adapters, experts, &d))
    return rc;
  XP_REQUIRE(dtype == XP_BFLOAT16 || dtype == XP_FLOAT16, "%s: type %d (bf16 or fp16)", what, dtype);
  XP_REQUIRE(K >= 8 && K % 8 == 0 && K <= (1 << 24) && n >= 8 && n % 8 == 0 && n <= (1 << 24),
             "%s: K=%lld and n=%lld must be positive multiples of 8", what, (long long)K, (long long)n);
  XP_REQUIRE(R == 16 || R == 32 || R == 64 || R == 96 || R == XP_LORA_MAX_RANK,
             "%s: storage rank %lld (16, 32, 64, 96 or %d)", what, (long long)R, XP_LORA_MAX_RANK);
  XP_REQUIRE(slices >= 1 && slices <= 16, "%s: %lld slices (1 to 16)", what, (long long)slices);
  if (T == 0) return XP_OK;
  const int64_t npairs = T * topk;
  const int64_t rows = per_pair ? npairs : T;
  XP_REQUIRE(x && a && b && scales && ranks && out, "%s: null argument", what);
  XP_REQUIRE(aligned16(x) && aligned16(a) && aligned16(b) && aligned16(out) && aligned16(base),
             "%s: buffers must be 16-byte aligned", what);
  XP_REQUIRE(x_stride % 8 == 0 && out_stride % 8 == 0 && base_stride % 8 == 0 && (x_stride >= K || rows <= 1) &&
                 (out_stride >= slices * n || npairs <= 1) && (!base || base_stride >= slices * n || npairs <= 1),
             "%s: row strides %lld, %lld and %lld must be multiples of 8 that hold a row", what, (long long)x_stride,
             (long long)base_stride, (long long)out_stride);
  const bool direct = npairs <= kDirectPairs;
  Listing w{nullptr, nullptr};
  if (!direct) {
    if (int rc = check_listing(what, npairs, adapters, experts, work, work_bytes)) return rc;
    listing_layout(npairs, adapters, experts, &w, static_cast<uint8_t*>(work));
    if (!grouped)
      if (int rc = launch_group(d, npairs, work, stream)) return rc;
  }
  Apply p{};
  p.x = static_cast<const uint16_t*>(x);
  p.x_stride = x_stride;
  p.per_pair = per_pair != 0;
  p.K = K;
  p.Kp = (K + 31) / 32 * 32;
  p.a = static_cast<const uint16_t*>(a);
  p.b = static_cast<const uint16_t*>(b);
  p.scales = scales;
  p.ranks = ranks;
  p.slices = static_cast<int>(slices);
  p.n = static_cast<int>(n);
  p.np = static_cast<int>((n + 15) / 16 * 16);
  p.base = static_cast<const uint16_t*>(base);
  p.base_stride = base_stride;
  p.out = static_cast<uint16_t*>(out);
  p.out_stride = out_stride;
  p.npairs = npairs;
  p.nsplit = 1;
  p.tiles = static_cast<int>(direct ? npairs : tile_places(npairs, adapters, experts));
  const int64_t grid = (p.tiles + 7) / 8 * 8 * slices * p.nsplit;
  XP_REQUIRE(grid <= INT32_MAX, "%s: %lld workgroups exceed the launch grid", what, (long long)grid);
  auto go = [&](auto* kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, as_stream(stream), d, p, w.pairs,
                       w.tiles);
  };
  auto by_type = [&](auto type) {
    using V = decltype(type);
    switch (R) {
      case 16: return go(lora_kernel<V, 1, 1>);
      case 32: return go(lora_kernel<V, 2, 1>);
      case 64: return go(lora_kernel<V, 4, 1>);
      case 96: return go(lora_kernel<V, 6, 1>);
      default: return go(lora_kernel<V, 8, 1>);
    }
  };
  if (dtype == XP_BFLOAT16)
    by_type(Bf16{});
  else
    by_type(Fp16{});
  return check_launch("lora_kernel");
}

}  // extern "C"

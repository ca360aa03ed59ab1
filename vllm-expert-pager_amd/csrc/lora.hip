// Low-rank adapters of many requests beside the experts' projections.
//
// Pair p = (token t, choice k) has the adapter of its token's request and the
// expert of its choice. Its row of a projection gets
//   scale B (A x)        A: [R][K], B: [n][R] of that (adapter, expert)
// per slice (gate and up are two slices with matrices of their own).
//
// The pairs of one (adapter, expert), a group, are multiplied together, a tile
// of up to 16 or 64 of them at a time: u = A x, K split over the workgroup's
// waves and summed in LDS, then B u over the workgroup's columns, with the
// 16x16x32 matrix instruction, the matrices as its first operand. Both products
// are one launch: a workgroup has its tile's u whole, and nothing but the
// result goes to memory. Bound by the bytes of A and B (with the top-k of
// hundreds of experts a group has few pairs) and of the result.
//
// Few tiles (decode steps): a workgroup per tile, slice and part of the
// columns, each of which makes u for itself from a matrix A that the parts
// read out of one L2 (64 dense tokens, rank 64: 13.7 us). Many tiles: a workgroup
// per tile of 64 pairs, as many of them at a time as its registers hold (MT
// fragments), and both slices of an even number where the rank is at most 32. A
// and B are read once for the tile at rank 16 and, for one slice, 32; twice at 64
// and for two slices of 32; at 96 and 128 once per 16 pairs. x is read once for
// the slices that go together (gate and up of 8192 tokens x 8, rank 16: 117 us,
// 617 MB at 5.2 TB/s).
//
// u enters the second product as the sum of two values of the operands' type,
// its rounding and the rounding of what is left, so no more than 2^-16 of it
// is lost (one rounding to bf16 would lose 2^-9). fp16 covers 2^-14 to 2^16
// with full precision, so there a pair's u is first scaled by a power of two
// that puts its largest value near 2^13, and the result scaled back.
//
// Grouping. Up to 64 pairs every wave groups them itself, up to 256 a workgroup
// finds the pairs of the same group as the one that its tile is named after.
// More pairs: a launch that sorts every 256 of them by range of groups, and one
// of a workgroup per range, which counts and places the groups of its range. A
// tile's place needs no count of the tiles before it: with tiles of n pairs, a
// range with pb pairs and gb groups below it starts at pb / n + min(gb, pb),
// which leaves room for its tiles whatever their sizes; unused places are
// marked empty.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <type_traits>

#include "common.h"

namespace xp {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kFrag = 16;             // pairs of a matrix instruction
constexpr int kWideTile = 64;         // pairs per tile where there are many
constexpr int kBallotPairs = 64;      // pairs that a wave groups
// Pairs that a workgroup groups, one a thread (of the 256 that the smaller form
// has). 32 tokens' down x 8 with eight adapters: 7.3 us, 18.2 by a listing; 128
// dense tokens of eight adapters: 17.4 and 19.1.
constexpr int kDirectPairs = 256;
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

// n / d for 0 <= n < 2^32 by a multiplication: with m = floor(2^64 / d) + 1 the
// product's high word is the quotient (a division is some 40 instructions).
struct Divisor {
  uint64_t m;  // 0: d = 1
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
    if (m == 0) return n;
    const uint64_t hi = static_cast<uint64_t>(n) * (m >> 32);
    return static_cast<uint32_t>((hi + __umulhi(n, static_cast<uint32_t>(m))) >> 32);
  }
};
inline Divisor divisor(int64_t d) { return Divisor{d == 1 ? 0 : ~0ull / static_cast<uint64_t>(d) + 1}; }

struct Ids {
  const void* adapter;
  const void* expert;  // null: expert 0
  int aeb, eeb;
  const int32_t* expert_map;  // null: every pair is listed
  int slots;
  int adapters, experts;
  Divisor by_topk, by_experts;
};

// Pair p's group: adapter * experts + expert, adapters * experts for a pair
// without an adapter, -1 for one that is not listed.
__device__ __forceinline__ int pair_group(const Ids& d, int64_t p) {
  const int64_t e = d.expert ? load_id(d.expert, d.eeb, p) : 0;
  const int64_t a = load_id(d.adapter, d.aeb, d.by_topk(static_cast<uint32_t>(p)));
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

// atomicAdd(&cell[g], 1) for the active lanes, those of the first lane's g in one
// addition: the pairs without an adapter, or a dense projection's, are one
// group of thousands, and 64 additions to one LDS word take 64 turns. Returns
// the lane's own place.
__device__ __forceinline__ int add_one(int* cell, int g) {
  const int g0 = __builtin_amdgcn_readfirstlane(g);
  const unsigned long long same = __ballot(g == g0);
  const int lead = __ffsll(static_cast<long long>(same)) - 1;
  int at = 0;
  if (g != g0 || static_cast<int>(threadIdx.x & 63) == lead) at = atomicAdd(&cell[g], g == g0 ? __popcll(same) : 1);
  const int base = __builtin_amdgcn_readlane(at, lead);
  return g == g0 ? base + static_cast<int>(lane_prefix(same)) : at;
}

// A chunk of kChunk pairs: (group, pair) by range of groups, in any order
// within a range, and where each range begins.
constexpr int kChunk = 256;
constexpr int kRanges = 256;  // ranges of groups, at most: the workgroups of group_kernel

__global__ void __launch_bounds__(kChunk) chunk_kernel(Ids d, int npairs, int per, int ranges,
                                                       int2* __restrict__ sorted, int32_t* __restrict__ starts) {
  __shared__ int s_count[kRanges];
  __shared__ int s_wave[kChunk / 64];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  s_count[tid] = 0;
  __syncthreads();
  const int p = blockIdx.x * kChunk + tid;
  const int g = p < npairs ? pair_group(d, p) : -1;
  const int r = g >= 0 ? static_cast<int>(static_cast<unsigned>(g) / static_cast<unsigned>(per)) : 0;
  int rank = 0;
  if (g >= 0) rank = add_one(s_count, r);
  __syncthreads();
  const int mine = s_count[tid];
  int in = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int v = __shfl_up(in, off, 64);
    if (lane >= off) in += v;
  }
  if (lane == 63) s_wave[wave] = in;
  __syncthreads();
  int before = in - mine;
  for (int w = 0; w < wave; ++w) before += s_wave[w];
  s_count[tid] = before;
  int32_t* row = starts + static_cast<int64_t>(blockIdx.x) * (ranges + 1);
  if (tid < ranges) row[tid] = before;
  if (tid == kRanges - 1) row[ranges] = before + mine;
  __syncthreads();
  if (g >= 0) sorted[static_cast<int64_t>(blockIdx.x) * kChunk + s_count[r] + rank] = make_int2(g, p);
}

// Workgroup w lists the groups [w per, (w + 1) per): pairs[] by group, and a
// tile entry per `tile` pairs of a group. It reads its range's part of every
// chunk, 16 lanes a chunk, twice (to count, and to place). The starts of the
// range in the chunks add up to the pairs of the ranges below. (Reading every
// pair's group in every workgroup took 34 to 90 us for 65536 pairs, however the
// own ones were taken out; a CU does not get through so many.)
__global__ void __launch_bounds__(kGroupThreads) group_kernel(const int2* __restrict__ sorted,
                                                              const int32_t* __restrict__ starts, int64_t npairs,
                                                              int groups, int per, int ranges, int tile,
                                                              int32_t* __restrict__ pairs,
                                                              Entry* __restrict__ tiles) {
  constexpr int kEach = kRangeGroups / kGroupThreads;
  constexpr int kTeam = 16, kTeams = kGroupThreads / kTeam;
  __shared__ int s_count[kRangeGroups];
  __shared__ int s_begin[kRangeGroups + 1], s_tile[kRangeGroups];  // a group's first pair and tile
  __shared__ int2 s_tot[kGroupThreads / 64];
  __shared__ int s_below, s_own;
  const int tid = threadIdx.x;
  const int g0 = blockIdx.x * per, g1 = g0 + per < groups ? g0 + per : groups;
  for (int i = tid; i < per; i += kGroupThreads) s_count[i] = 0;
  if (tid == 0) s_below = s_own = 0;
  __syncthreads();
  const int own_groups = g1 > g0 ? g1 - g0 : 0;
  const int nchunk = static_cast<int>((npairs + kChunk - 1) / kChunk);
  // The range's pairs, a team of kTeam lanes a chunk and kRound chunks of a team
  // at a time, so that their starts, and then their first pairs, are requested
  // together. One round covers 65536 pairs, and its pairs stay in registers.
  constexpr int kRound = 4;
  const int lane16 = tid % kTeam;
  int lo[kRound], hi[kRound];
  int2 v[kRound];
  auto chunk_of = [&](int c0, int i) { return c0 + tid / kTeam + i * kTeams; };
  auto load_round = [&](int c0) {
#pragma unroll
    for (int i = 0; i < kRound; ++i) {
      const int c = chunk_of(c0, i);
      lo[i] = hi[i] = 0;
      if (c < nchunk) {
        const int32_t* row = starts + static_cast<int64_t>(c) * (ranges + 1) + blockIdx.x;
        lo[i] = row[0];
        hi[i] = row[1];
      }
    }
#pragma unroll
    for (int i = 0; i < kRound; ++i)
      if (lo[i] + lane16 < hi[i]) v[i] = sorted[static_cast<int64_t>(chunk_of(c0, i)) * kChunk + lo[i] + lane16];
  };
  auto each_pair = [&](int c0, auto&& f) {
#pragma unroll
    for (int i = 0; i < kRound; ++i) {
      if (lo[i] + lane16 < hi[i]) f(v[i]);
      for (int k = lo[i] + lane16 + kTeam; k < hi[i]; k += kTeam)
        f(sorted[static_cast<int64_t>(chunk_of(c0, i)) * kChunk + k]);
    }
  };
  const bool once = nchunk <= kRound * kTeams;
  int below = 0, own = 0;
  for (int c0 = 0; c0 < nchunk; c0 += kRound * kTeams) {
    load_round(c0);
#pragma unroll
    for (int i = 0; i < kRound; ++i) {
      below += lo[i];
      own += hi[i] - lo[i];
    }
    each_pair(c0, [&](int2 p) { add_one(s_count, p.x - g0); });
  }
  if (tid % kTeam == 0 && (below | own)) {
    atomicAdd(&s_below, below);
    atomicAdd(&s_own, own);
  }
  __syncthreads();
  const int pb = s_below;
  own = s_own;
  // A thread's kEach consecutive groups: first pair and first tile.
  int c[kEach];
  int2 mine = make_int2(0, 0);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int g = tid * kEach + i;
    c[i] = g < own_groups ? s_count[g] : 0;
    mine.x += c[i];
    mine.y += (c[i] + tile - 1) / tile;
  }
  int2 at = block_scan2(mine, s_tot);  // (a barrier: the counts are read)
  const int first = pb / tile + (g0 < pb ? g0 : pb);
  const int upto = g0 + own_groups, pe = pb + own;
  const int last = pe / tile + (upto < pe ? upto : pe);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int g = tid * kEach + i;
    if (g < own_groups) {
      s_count[g] = pb + at.x;  // where the group's next pair goes
      s_begin[g] = pb + at.x;
      s_tile[g] = at.y;
    }
    at.x += c[i];
    at.y += (c[i] + tile - 1) / tile;
  }
  if (tid == 0) s_begin[own_groups] = pe;
  __syncthreads();
  int used = 0;
  for (int w = 0; w < kGroupThreads / 64; ++w) used += s_tot[w].y;
  // Tile t belongs to the last group whose tiles begin at or before it.
  for (int t = tid; t < used; t += kGroupThreads) {
    int a = 0, z = own_groups;
    while (z - a > 1) {
      const int m = (a + z) >> 1;
      if (s_tile[m] <= t)
        a = m;
      else
        z = m;
    }
    const int from = s_begin[a] + (t - s_tile[a]) * tile, left = s_begin[a + 1] - from;
    tiles[first + t] = Entry{g0 + a, from, left < tile ? left : tile, 0};
  }
  for (int i = first + used + tid; i < last; i += kGroupThreads) tiles[i] = Entry{0, 0, 0, 0};
  // The places behind the last range, by the last workgroup.
  if (blockIdx.x == gridDim.x - 1) {
    const int64_t bound = npairs / tile + (groups < npairs ? groups : npairs);
    for (int64_t i = last + tid; i < bound; i += kGroupThreads) tiles[i] = Entry{0, 0, 0, 0};
  }
  for (int c0 = 0; c0 < nchunk; c0 += kRound * kTeams) {
    if (!once) load_round(c0);
    each_pair(c0, [&](int2 p) {
      const int at = add_one(s_count, p.x - g0);
      pairs[at] = p.y;
    });
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

// Tile i of up to kBallotPairs pairs, by every wave for itself, a pair a lane:
// the lanes of one group are found bit by bit, and the tiles numbered in the
// order of the groups' first pairs, so that the first places are the live ones.
// Returns the pairs' number (0: no such tile), row r's pair in lane r.
__device__ __forceinline__ int ballot_tile(const Ids& d, int npairs, int i, int& group, int& row_pair) {
  const int lane = threadIdx.x & 63;
  const int g = lane < npairs ? pair_group(d, lane) : -1;
  unsigned long long same = __ballot(g >= 0);
  const int bits = 32 - __clz(d.adapters * d.experts);
#pragma unroll 1
  for (int b = 0; b < bits; ++b) {
    const bool set = (g >> b) & 1;
    const unsigned long long m = __ballot(set);
    same &= set ? m : ~m;
  }
  const int rank = static_cast<int>(lane_prefix(same));
  const int ntile = g >= 0 && rank == 0 ? (__popcll(same) + kFrag - 1) / kFrag : 0;
  int start = 0;
#pragma unroll
  for (int b = 0; b < 3; ++b) start += static_cast<int>(lane_prefix(__ballot((ntile >> b) & 1))) << b;
  const unsigned long long own = __ballot(ntile > 0 && start <= i && i < start + ntile);
  if (own == 0) return 0;
  const int lead = __ffsll(static_cast<long long>(own)) - 1;
  group = __builtin_amdgcn_readlane(g, lead);
  const int r0 = (i - __builtin_amdgcn_readlane(start, lead)) * kFrag;
  const int all = __popcll(__ballot(g == group));
  const int r = rank - r0;
  const bool in = g == group && r >= 0 && r < kFrag;
  // Row r's pair goes to lane r; the other lanes' go to lane 63.
  row_pair = __builtin_amdgcn_ds_permute(4 * (in ? r : 63), lane);
  return all - r0 < kFrag ? all - r0 : kFrag;
}

// Tile i of more pairs, up to kDirectPairs, by the whole workgroup (a thread
// per pair at least): the tile of pair i, if i is the first, the 17th, ... pair
// of its group. Only that group matters, so one comparison a thread finds its
// pairs. (Numbering the tiles took 46 LDS reads a thread for 184 pairs, and 5.2
// us of 14.) Returns the pairs' number (0: no such tile); the barrier behind
// s_pair is the caller's.
__device__ __forceinline__ int direct_tile(const Ids& d, int npairs, int i, unsigned long long* s_mask, int* s_pair,
                                           int& group) {
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  group = pair_group(d, i);
  const int g = tid < npairs ? pair_group(d, tid) : -1;
  const unsigned long long mine = __ballot(g == group && g >= 0);
  if (lane == 0 && wave < kDirectPairs / 64) s_mask[wave] = mine;
  if (tid < kFrag) s_pair[tid] = i;  // rows past the count repeat the first
  __syncthreads();
  int before = 0, total = 0, own = static_cast<int>(lane_prefix(mine));
#pragma unroll
  for (int w = 0; w < kDirectPairs / 64; ++w) {
    const unsigned long long m = s_mask[w];
    const int n = __popcll(m);
    if (w < (i >> 6)) before += n;
    if (w == (i >> 6)) before += __popcll(m & ((1ull << (i & 63)) - 1));
    if (w < wave) own += n;
    total += n;
  }
  if (group < 0 || before % kFrag != 0) return 0;
  const int r = own - before;
  if (g == group && r > 0 && r < kFrag) s_pair[r] = tid;
  return total - before < kFrag ? total - before : kFrag;
}

// RB: 16-row blocks of a slice's rank. SPW: slices per workgroup. MT: 16-pair
// fragments multiplied at a time. NW: waves.
template <typename T, int RB, int SPW, int MT, int NW>
__global__ void __launch_bounds__(64 * NW, MT == 1 ? 2 : 3) lora_kernel(Ids d, Apply p, const int32_t* __restrict__ pairs,
                                                       const Entry* __restrict__ tiles) {
  constexpr int NB = RB * SPW, R = 16 * RB, NT = 64 * NW;
  constexpr int kRow = R + 8;   // an LDS row of u: 16 bytes more, so that the rows spread over the banks
  // K steps whose loads are in flight together. With few tiles a CU has one
  // workgroup, whose latencies count and whose registers do not: all its loads
  // at once, and B's first rows requested before u is made.
  constexpr bool kFew = MT == 1;
  constexpr int kAhead = kFew ? (NB > 6 ? 2 : NB > 2 ? 4 : 8) : (NB + MT > 6 ? 1 : NB + MT > 3 ? 2 : 4);
  static_assert(NT >= kDirectPairs, "a thread per pair that is grouped here");
  __shared__ int s_pair[kWideTile];
  __shared__ unsigned long long s_mask[kDirectPairs / 64];
  __shared__ __attribute__((aligned(16))) float s_u[NW][NB * MT][kFrag][16];
  __shared__ __attribute__((aligned(16))) uint16_t s_hi[SPW][MT * kFrag][kRow], s_lo[SPW][MT * kFrag][kRow];
  __shared__ float s_back[SPW][MT * kFrag];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4, j = lane & 15;
  // Workgroups go to the XCDs in turn, and the grid's width is a multiple of
  // 8: a tile's parts (slices, columns) read its matrices into one L2.
  // Listed tiles are dealt in runs of kRun, so that a group's tiles mostly read
  // its matrices into one as well (8192 tokens' gate and up: 642 MB moved dealt
  // one by one, of which 93 are A again; 120 -> 115 us at best).
  constexpr int kRun = 4;
  const int at = blockIdx.x >> 3;
  const int ti = pairs ? (at / kRun * 8 + (blockIdx.x & 7)) * kRun + at % kRun : static_cast<int>(blockIdx.x);
  if (ti >= p.tiles) return;
  const int s0 = blockIdx.z * SPW, split = blockIdx.y;

  int group, count;
  if (pairs) {
    const Entry e = tiles[ti];
    // (a listing of other sizes addresses nothing out of range)
    if (e.count <= 0 || e.count > kWideTile || e.first < 0 || e.first + e.count > p.npairs || e.group < 0 ||
        e.group > d.adapters * d.experts)
      return;
    group = e.group;
    count = e.count;
    if (tid < kWideTile) {
      const int pr = pairs[e.first + (tid < count ? tid : 0)];
      s_pair[tid] = pr < 0 ? 0 : (pr < p.npairs ? pr : static_cast<int>(p.npairs - 1));
    }
  } else {
    if (p.npairs <= kBallotPairs) {
      int row_pair;
      count = ballot_tile(d, static_cast<int>(p.npairs), ti, group, row_pair);
      const int first = __builtin_amdgcn_readlane(row_pair, 0);
      if (tid < kFrag) s_pair[tid] = tid < count ? row_pair : first;
    } else {
      count = direct_tile(d, static_cast<int>(p.npairs), ti, s_mask, s_pair, group);
    }
    if (count == 0) return;
  }
  group = __builtin_amdgcn_readfirstlane(group);
  count = __builtin_amdgcn_readfirstlane(count);

  // This workgroup's 32-column blocks of a slice.
  const int blocks = p.np / 32, per_split = (blocks + p.nsplit - 1) / p.nsplit;
  const int b0 = split * per_split, b1 = b0 + per_split < blocks ? b0 + per_split : blocks;

  if (group == d.adapters * d.experts) {  // no adapter: base, or zeros
    if (p.out == p.base) return;
    __syncthreads();
    const int c0 = b0 * 4, c1 = (b1 * 32 < p.n ? b1 * 32 : p.n) / 8;  // 8-column pieces
    for (int s = s0; s < s0 + SPW; ++s)
      for (int i = tid; i < count * (c1 - c0); i += NT) {
        const int r = i / (c1 - c0), c = s * p.n + (c0 + i - r * (c1 - c0)) * 8;
        const int64_t pr = s_pair[r];
        u32x4 v = {0, 0, 0, 0};
        if (p.base) v = *reinterpret_cast<const u32x4*>(p.base + pr * p.base_stride + c);
        *reinterpret_cast<u32x4*>(p.out + pr * p.out_stride + c) = v;
      }
    return;
  }
  const int adapter = __builtin_amdgcn_readfirstlane(static_cast<int>(d.by_experts(group)));
  int rank = p.ranks[adapter];
  rank = rank < 0 ? 0 : (rank < R ? rank : R);
  const int live = (rank + 15) / 16;  // 16-row blocks of a slice that hold anything
  const float scale = p.scales[adapter];
  const int steps = static_cast<int>(p.Kp / 32);
  // A's 16 x 32 blocks lie one behind the other in lane order: a load is 1 KB
  // in a row. (By rows of K values, 16 rows 4 KB apart are all in one channel
  // of the L2.)
  // B's rows of 32 columns, kBlocks blocks of a wave at a time, the first ones
  // requested before u is made.
  constexpr int KS = RB == 1 ? 1 : RB / 2;
  constexpr int kBlocks = RB == 1 && SPW == 1 && !kFew ? 8 : KS == 1 ? 4 : KS == 2 ? 2 : 1;
  // RB = 1: a row is 32 bytes, half an instruction's; the lanes of the upper half
  // load the second instruction's rows, and the halves are exchanged where they
  // are used, so that a load has no row twice (2048 tokens' down 50 -> 46 us).
  constexpr int kHalves = RB == 1 ? 1 : 2;
  u32x4 bv[kBlocks][kHalves][KS];
  auto load_b = [&](int s, int blk0) {
    const uint16_t* bmat = p.b + (static_cast<int64_t>(group) * p.slices + s0 + s) * p.np * R;
    // (an offset of the lane in 32 bits, everything else the same for the wave)
    const uint32_t own =
        RB == 1 ? (8 * (j >> 2) + (j & 3) + 4 * (q >> 1)) * R + 8 * (q & 1) : (8 * (j >> 2) + (j & 3)) * R + 8 * q;
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      const int blk = __builtin_amdgcn_readfirstlane(blk0 + i * NW < b1 ? blk0 + i * NW : b1 - 1);
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int k = 0; k < KS; ++k)
          if (KS == 1 || 32 * k < rank)
            bv[i][h][k] =
                *reinterpret_cast<const u32x4*>(bmat + static_cast<int64_t>(32 * blk + 4 * h) * R + 32 * k + own);
    }
  };
  const uint16_t* ablk = p.a + (static_cast<int64_t>(group) * p.slices + s0) * R * p.Kp;
  const uint32_t alane = 8 * lane;

#pragma unroll 1
  for (int m0 = 0; m0 < count; m0 += MT * kFrag) {
    const int frags = count - m0 < MT * kFrag ? (count - m0 + kFrag - 1) / kFrag : MT;
    // u = A x: wave w takes the K steps w, w + NW, ..., kAhead of them at a
    // time, the rows of A (which need no pair) requested first.
    f32x4 acc[NB][MT];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[i][m] = f32x4{0.f, 0.f, 0.f, 0.f};
    const uint16_t* xrow[MT];
    if (kFew && b0 < b1) load_b(0, b0 + wave);
#pragma unroll 1
    for (int k0 = wave; k0 < steps; k0 += NW * kAhead) {
      u32x4 av[kAhead][NB], xv[kAhead][MT];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int k = k0 + u * NW;
        if (k >= steps) continue;
#pragma unroll
        for (int i = 0; i < NB; ++i)  // (a block past the rank reads zeros that nothing uses)
          if (RB <= 2 || i % RB < live)
            av[u][i] = *reinterpret_cast<const u32x4*>(ablk + (static_cast<int64_t>(i) * steps + k) * 512 + alane);
      }
      if (k0 == wave) {
        if (m0 == 0) __syncthreads();  // s_pair
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const int pr = s_pair[m0 + (m < frags ? m : 0) * kFrag + j];
          xrow[m] = p.x + static_cast<int64_t>(p.per_pair ? pr : d.by_topk(pr)) * p.x_stride + 8 * q;
        }
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int k = k0 + u * NW;
        if (k >= steps) continue;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          xv[u][m] = u32x4{0, 0, 0, 0};
          if (m < frags && 32 * k + 8 * q < p.K) xv[u][m] = *reinterpret_cast<const u32x4*>(xrow[m] + 32 * k);
        }
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (k0 + u * NW >= steps) continue;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          if (RB > 2 && i % RB >= live) continue;
#pragma unroll
          for (int m = 0; m < MT; ++m)
            if (m < frags) acc[i][m] = T::mfma(av[u][i], xv[u][m], acc[i][m]);
        }
      }
    }
    if (wave >= steps && m0 == 0) __syncthreads();  // a wave without a step meets the others at s_pair too
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int m = 0; m < MT; ++m) *reinterpret_cast<f32x4*>(&s_u[wave][i * MT + m][j][4 * q]) = acc[i][m];
    __syncthreads();
    // The waves' sums, and u in two values: 16 threads per pair.
    for (int sm = tid >> 8; sm < SPW * MT; sm += NT / 256) {
      const int s = sm / MT, m = sm % MT;
      const int pr = (tid >> 4) & 15, t16 = tid & 15;
      float u[RB];
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        float v = s_u[0][(s * RB + i) * MT + m][pr][t16];
#pragma unroll
        for (int w = 1; w < NW; ++w) v += s_u[w][(s * RB + i) * MT + m][pr][t16];
        u[i] = 16 * i + t16 < rank ? v : 0.0f;  // zero rows of A times an infinite x are not zero
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
      if (t16 == 0) s_back[s][m * kFrag + pr] = back;
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const float v = u[i] * up;
        const uint16_t hi = T::bits(v);
        const float rest = v - T::value(hi);
        s_hi[s][m * kFrag + pr][16 * i + t16] = hi;
        s_lo[s][m * kFrag + pr][16 * i + t16] = fabsf(T::value(hi)) < INFINITY ? T::bits(rest) : 0;
      }
    }
    __syncthreads();

    // B u for this workgroup's columns, 32 at a time: row i of the first of
    // the two instructions is column 8 (i / 4) + i % 4, of the second 4 more,
    // so that a lane's eight outputs are eight consecutive columns of a pair.
#pragma unroll
    for (int s = 0; s < SPW; ++s) {
      if (s > 0 || !kFew) load_b(s, b0 + wave);
      // RB = 1: the lanes of the upper half of the instruction's 32 take what
      // is left of u, with the same 16 columns of B.
      u32x4 hi[MT][KS], lo[MT][KS];
      float f[MT];
      int64_t row[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int r = m * kFrag + j;
        f[m] = scale * s_back[s][r];
        row[m] = s_pair[m0 + (m < frags ? r : j)];
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          if constexpr (RB == 1) {
            hi[m][0] = *reinterpret_cast<const u32x4*>(q < 2 ? &s_hi[s][r][8 * q] : &s_lo[s][r][8 * (q - 2)]);
          } else {
            hi[m][k] = *reinterpret_cast<const u32x4*>(&s_hi[s][r][32 * k + 8 * q]);
            lo[m][k] = *reinterpret_cast<const u32x4*>(&s_lo[s][r][32 * k + 8 * q]);
          }
        }
      }
#pragma unroll 1
      for (int blk0 = b0 + wave; blk0 < b1; blk0 += NW * kBlocks) {
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
          const int blk = blk0 + i * NW;
          if (blk >= b1) continue;
          const int c = 32 * blk + 8 * q;
          u32x4 bw[2][KS];
          if constexpr (RB == 1) {
            // Both halves of the wave get the lower half's rows, and the upper's.
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const auto t = __builtin_amdgcn_permlane32_swap(bv[i][0][0][w], bv[i][0][0][w], false, false);
              bw[0][0][w] = t[0];
              bw[1][0][w] = t[1];
            }
          } else {
#pragma unroll
            for (int k = 0; k < KS; ++k) {
              bw[0][k] = bv[i][0][k];
              bw[1][k] = bv[i][kHalves - 1][k];
            }
          }
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            if (m >= frags) continue;
            f32x4 y[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int k = 0; k < KS; ++k) {
                if (KS > 1 && 32 * k >= rank) continue;
                y[h] = T::mfma(bw[h][k], hi[m][k], y[h]);
                if constexpr (RB > 1) y[h] = T::mfma(bw[h][k], lo[m][k], y[h]);
              }
            if (m0 + m * kFrag + j >= count || c >= p.n) continue;
            const int64_t col = static_cast<int64_t>(s0 + s) * p.n + c;
            float v[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) v[r] = y[r >> 2][r & 3] * f[m];
            if (p.base) {
              const u32x4 w = *reinterpret_cast<const u32x4*>(p.base + row[m] * p.base_stride + col);
#pragma unroll
              for (int r = 0; r < 8; ++r) v[r] += T::value(static_cast<uint16_t>(w[r >> 1] >> (16 * (r & 1))));
            }
            u32x4 o;
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = T::bits(v[2 * r]) | static_cast<uint32_t>(T::bits(v[2 * r + 1])) << 16;
            *reinterpret_cast<u32x4*>(p.out + row[m] * p.out_stride + col) = o;
          }
        }
        if (blk0 + NW * kBlocks < b1) load_b(s, blk0 + NW * kBlocks);
      }
    }
    if (m0 + MT * kFrag < count) __syncthreads();  // s_u, s_hi and s_lo are written again
  }
}

// ---- host side ----

int64_t align256(int64_t n) { return (n + 255) & ~int64_t(255); }

// Pairs per tile of a listing: 64 where that still makes a tile or more for
// every CU, whether by the pairs or by the groups, else 16 (more workgroups).
// By the sizes alone, so that a listing serves every projection of a call. us
// with 64 and with 16: 1024 tokens x 4 of 32 experts (64 groups) 34 and 24, 2048
// dense tokens of four adapters 34 and 21; gate and up of 8192 tokens x 8 of 256
// experts with 2, 4, 8 and 16 adapters 96, 109, 132 and 187 and 136, 147, 164
// and 209, of 2048 tokens with one 32 and 39, with four 57 and 58.
int tile_pairs(int64_t npairs, int64_t adapters, int64_t experts) {
  return npairs / kWideTile >= 256 || std::min(adapters * experts, npairs) >= 256 ? kWideTile : kFrag;
}

// The same for a call that makes its own listing, which knows its projection: a
// single slice of rank 16 gains little from 64 (16 rows of A are soon read) and
// loses the workgroups. us with 64 and with 16, 256 experts x 8 and four
// adapters: K = 512, 2048 and 4096, 2048 tokens 46 and 41, 76 and 64, 105 and 86,
// 8192 tokens 122 and 117, 166 and 160, 223 and 208; 32768 dense tokens (2048 x
// 2048) of 16 adapters 84 and 76, of one 77 and 88. With rank 32 (K = 512, 8192
// tokens) 136 and 177, dense 96 and 111; rank 64 dense 135 and 191.
// Ranks 96 and 128 have no shape of more than 16 pairs at a time (pick_shape), so
// a tile of 64 reads A and B as often as four of 16, in a quarter of the
// workgroups: down of 2048 tokens with two adapters 160 and 105, 215 and 138, of
// 8192 with one 276 and 263, 421 and 365; gate and up of 8192 tokens x 4 of 64
// experts 211 and 169, 317 and 265; 32768 dense tokens of 16 adapters 219 and 177,
// 350 and 264, of one 151 and 153, 226 and 234.
int own_tile_pairs(int64_t npairs, int64_t adapters, int64_t experts, int64_t slices, int64_t R) {
  return R >= 96 || (R == 16 && slices % 2 == 1) ? kFrag : tile_pairs(npairs, adapters, experts);
}

// Workgroups that a call of few tiles is split into, about. Every part of a
// tile's columns reads A for itself: the parts share an L2, which gives about
// 20 CUs what each can take, so beyond some 160 workgroups they wait for it (64
// dense tokens of 24 adapters of rank 64: 13.8 us with 160, 23 with 256).
constexpr int64_t kFillWorkgroups = 160;
constexpr int64_t kPartBlocks = 2;        // 32-column blocks of a part, at least

// Places of the tile list: npairs / tile + min(groups, npairs), the group of
// the pairs without an adapter among them.
int64_t tile_places(int64_t npairs, int64_t adapters, int64_t experts, int tile) {
  return npairs / tile + std::min(adapters * experts + 1, npairs);
}

struct Listing {
  int2* sorted;     // [chunk][kChunk]
  int32_t* starts;  // [chunk][ranges + 1]
  int32_t* pairs;
  Entry* tiles;
};

// Groups per range, of at most kRanges ranges (at most kRangeGroups of the 2^20 groups).
int64_t range_groups(int64_t groups) { return (groups + kRanges - 1) / kRanges; }

int64_t listing_layout(int64_t npairs, int64_t adapters, int64_t experts, Listing* w, uint8_t* base) {
  const int64_t groups = adapters * experts + 1, per = range_groups(groups), ranges = (groups + per - 1) / per;
  const int64_t chunks = (npairs + kChunk - 1) / kChunk;
  const int64_t sz[4] = {align256(npairs * 8), align256(chunks * (ranges + 1) * 4), align256(npairs * 4),
                         align256(tile_places(npairs, adapters, experts, kFrag) * static_cast<int64_t>(sizeof(Entry)))};
  if (w) {
    w->sorted = reinterpret_cast<int2*>(base);
    w->starts = reinterpret_cast<int32_t*>(base + sz[0]);
    w->pairs = reinterpret_cast<int32_t*>(base + sz[0] + sz[1]);
    w->tiles = reinterpret_cast<Entry*>(base + sz[0] + sz[1] + sz[2]);
  }
  return sz[0] + sz[1] + sz[2] + sz[3];
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
  *d = Ids{adapter_ids, topk_ids, aeb, eb, expert_map, static_cast<int>(slots),
           static_cast<int>(adapters), static_cast<int>(experts), divisor(topk), divisor(experts)};
  return XP_OK;
}

int check_listing(const char* what, int64_t npairs, int64_t adapters, int64_t experts, const void* work, int64_t bytes) {
  const int64_t need = listing_layout(npairs, adapters, experts, nullptr, nullptr);
  XP_REQUIRE(work && (reinterpret_cast<uintptr_t>(work) & 255) == 0 && bytes >= need,
             "%s: the workspace must be 256-byte aligned and of %lld B", what, (long long)need);
  return XP_OK;
}

int launch_group(const Ids& d, int64_t npairs, int tile, void* work, void* stream) {
  Listing w;
  listing_layout(npairs, d.adapters, d.experts, &w, static_cast<uint8_t*>(work));
  const int64_t groups = static_cast<int64_t>(d.adapters) * d.experts + 1;
  const int per = static_cast<int>(range_groups(groups));
  const unsigned ranges = static_cast<unsigned>((groups + per - 1) / per);
  hipLaunchKernelGGL(chunk_kernel, dim3(static_cast<unsigned>((npairs + kChunk - 1) / kChunk)), dim3(kChunk), 0,
                     as_stream(stream), d, static_cast<int>(npairs), per, static_cast<int>(ranges), w.sorted, w.starts);
  if (int rc = check_launch("chunk_kernel")) return rc;
  hipLaunchKernelGGL(group_kernel, dim3(ranges), dim3(kGroupThreads), 0, as_stream(stream), w.sorted, w.starts, npairs,
                     static_cast<int>(groups), per, static_cast<int>(ranges), tile, w.pairs, w.tiles);
  return check_launch("group_kernel");
}

// One workgroup's shape for RB 16-row blocks of rank: with many tiles MT
// fragments and, where the slices allow, two slices, as many as a workgroup's
// LDS and registers hold (8 sums of 16 x 16); with few, one of each and eight
// waves, so that K is split further.
template <typename T, int RB, typename F>
void pick_shape(bool wide, bool even, F&& go) {
  constexpr int few = RB <= 4 ? 8 : 4;
  if constexpr (RB == 1) {
    if (wide) return even ? go(lora_kernel<T, 1, 2, 4, 4>, 2, 4) : go(lora_kernel<T, 1, 1, 4, 4>, 1, 4);
  } else if constexpr (RB == 2) {
    if (wide) return even ? go(lora_kernel<T, 2, 2, 2, 4>, 2, 4) : go(lora_kernel<T, 2, 1, 4, 4>, 1, 4);
  } else if constexpr (RB == 4) {
    if (wide) return go(lora_kernel<T, 4, 1, 2, 4>, 1, 4);
  }
  return go(lora_kernel<T, RB, 1, 1, few>, 1, few);
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
  return launch_group(d, T * topk, tile_pairs(T * topk, adapters, experts), work, stream);
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
  XP_REQUIRE(out != base || base_stride == out_stride || npairs <= 1,
             "%s: rows of out and base, in one place, are %lld and %lld elements apart", what, (long long)out_stride,
             (long long)base_stride);
  const bool direct = npairs <= kDirectPairs;
  const int tile = direct    ? kFrag
                   : grouped ? tile_pairs(npairs, adapters, experts)
                             : own_tile_pairs(npairs, adapters, experts, slices, R);
  Listing w{};
  if (!direct) {
    if (int rc = check_listing(what, npairs, adapters, experts, work, work_bytes)) return rc;
    listing_layout(npairs, adapters, experts, &w, static_cast<uint8_t*>(work));
    if (!grouped)
      if (int rc = launch_group(d, npairs, tile, work, stream)) return rc;
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
  p.np = static_cast<int>((n + 31) / 32 * 32);
  p.base = static_cast<const uint16_t*>(base);
  p.base_stride = base_stride;
  p.out = static_cast<uint16_t*>(out);
  p.out_stride = out_stride;
  p.npairs = npairs;
  p.tiles = static_cast<int>(direct ? npairs : tile_places(npairs, adapters, experts, tile));
  // The tiles that can be there: parts of the columns for the rest of the CUs.
  const bool wide = tile == kWideTile;
  const int64_t likely = std::max(npairs / (wide ? kWideTile : kFrag), std::min(adapters * experts, npairs));
  int rc = XP_OK;
  auto launch = [&](auto* kernel, int spw, int waves) {
    const int64_t fill = kFillWorkgroups / std::max<int64_t>(1, likely * (slices / spw));
    p.nsplit = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(fill, p.np / 32 / kPartBlocks)));
    const int round = direct ? 8 : 32;  // the XCDs, and runs of four tiles for each
    const dim3 grid(static_cast<unsigned>((p.tiles + round - 1) / round * round), static_cast<unsigned>(p.nsplit),
                    static_cast<unsigned>(slices / spw));
    if (static_cast<int64_t>(grid.x) * 64 * waves > UINT32_MAX) {
      rc = fail(XP_E_LIMIT, "%s: %lld pairs exceed the launch grid", what, (long long)npairs);
      return;
    }
    hipLaunchKernelGGL(kernel, grid, dim3(static_cast<unsigned>(64 * waves)), 0, as_stream(stream), d, p, w.pairs,
                       w.tiles);
    rc = check_launch("lora_kernel");
  };
  auto by_type = [&](auto type) {
    using V = decltype(type);
    const bool even = slices % 2 == 0;
    switch (R) {
      case 16: return pick_shape<V, 1>(wide, even, launch);
      case 32: return pick_shape<V, 2>(wide, even, launch);
      case 64: return pick_shape<V, 4>(wide, even, launch);
      case 96: return pick_shape<V, 6>(wide, even, launch);
      default: return pick_shape<V, 8>(wide, even, launch);
    }
  };
  if (dtype == XP_BFLOAT16)
    by_type(Bf16{});
  else
    by_type(Fp16{});
  return rc;
}

}  // extern "C"

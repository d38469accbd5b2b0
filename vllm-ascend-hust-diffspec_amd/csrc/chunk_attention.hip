// Attention of a chunk of new tokens over a paged cache.
//
// Prompts enter a serving engine in chunks: ragged rows of query tokens (query_start, query_len),
// the last of their target_len tokens, attend over their pages (block_table); rows that decode a
// single token ride in the same batch.  With
//
//   L(b, i) = target_len[b] - query_len[b] + i + 1     keys before and at query token i of row b
//
// query token i sees the keys max(0, L - window) <= t < L, and
//
//   out = sum_t softmax_t(scale q . k_t) v_t,  lse = ln sum_t exp(scale q . k_t).
//
// The query heads that share a KV head are rows of one matrix (row = token * group + head in the
// group).  An item is 128 of a row's matrix rows over the keys that they see, for every KV head; items
// of many key tiles are cut into parts of nearly one size, whose pieces (maximum, sum, output, in fp32)
// chunk_join_kernel puts together.  chunk_plan_kernel derives items and parts from the lengths on the
// device, so that a captured launch follows changed lengths, and lists them by size, the largest first.
//
// Each of four waves has 32 query rows as columns of the score product, so that a lane's scores are of one row and the
// weights are in the layout that the second product takes; tiles of 64 keys go by in shared memory for all
// four.  What bounds it: vector instructions beside the matrix units (about 240 a wave and tile, 32 of them exponentials,
// against 32 products of 32 cycles at 128 dimensions: 58% and 46% of the cycles), and at 256 dimensions that a SIMD has
// registers for one wave only, which waits for a third of its cycles.  Measured,
// 32 query heads on 8 of 128 dimensions: 4096 tokens on themselves 167 us (823 TFLOP/s), of which the plan and a join
// with nothing to join take 8 to 10;
// 32 on 4, 512 tokens on 32 k keys 292 us (935); 11 mixed requests, 64 heads on 8 of 64 dimensions, 102 us (518); 3 chunks
// of 16 heads on 2 of 256 dimensions, window 1024, 181 us (530); 37 tokens 19.8 us.  A large library product reaches 1273.
#include <cmath>
#include <type_traits>

#include "matrix.h"

namespace ds355 {
namespace {

constexpr int kItemRows = 128;  // query rows of an item
// Key tiles below which an item is not cut.  A part waits for its first tile, and pieces have to be joined: 37 tokens on
// 248 keys take 19.3 us with 4 and 18.2 with 1 or 2, 128 on 1 k 25.3 and 34.8 with 1, 27.1 with 2, 28.1 with 8, eight single
// tokens on 500 keys 19.6 and 18.7 with 2, 23.2 with 8; a single token on 32 k 81 and 61 with 8, whose pieces are fewer.
constexpr int kMinPart = 4;
constexpr uint32_t kStatusRow = 1;     // a row's query tokens are out of range
constexpr uint32_t kStatusLength = 2;  // a row is longer than its block table
constexpr uint32_t kStatusPage = 4;    // a page id is out of range

constexpr int kTile = 64;  // keys of a staged tile
constexpr int kScores = kTile / 32;  // score products of a wave's tile
// As many as fit: a wave's outputs and queries take 48, 96 or 192 registers (162, 229 and, with accumulation registers, 432 in
// all), and the tiles 32, 64 or 128 KiB of shared memory.
constexpr int chunk_waves(int d) { return d == 64 ? 3 : d == 128 ? 2 : 1; }  // workgroups of a CU, waves of a SIMD
int part_slots(int d) { return chunk_waves(d) * device_cu_count(); }  // workgroups that run at a time

template <int D>
struct Chunk {
  static constexpr int kWaves = 4;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kPieces = D / 8;  // 16-byte pieces of a key
  static constexpr int kStage = kTile * kRowBytes;  // bytes of a tile's keys, or of its values
  static constexpr int kSteps = D / 16;   // score products of 32 keys
  static constexpr int kBlocks = D / 32;  // output blocks of 32 dimensions
  static constexpr int kPerLoad = 64 / kPieces;               // keys that one load of a wave covers
  static constexpr int kLoads = kTile / kPerLoad / kWaves;    // such loads of a wave for the keys of a tile
};

// An entry of the plan: one part of an item, the same for every KV head.
struct Part {
  int start, len, seen;  // the row's first query token, its query tokens, the keys before its first one
  int row, tile;         // row of the batch, 128 query rows of it
  int part, parts;       // which of the item's parts
  int slot;              // its first piece, in units of KV heads
};
static_assert(sizeof(Part) == 32);

struct PlanHeader {
  int parts, joins;
  int unused[62];
  int zeros[64];  // what keys past an item's end and those of a page out of range are read from
};

struct ChunkArgs {
  const uint16_t* q;
  int64_t q_row, q_head;
  uint16_t* out;
  int64_t o_row, o_head;
  float* lse;
  int64_t l_row, l_head;
  const char* k;
  int64_t k_block, k_token, k_head;  // bytes
  const char* v;
  int64_t v_block, v_token, v_head;
  const int32_t* table;
  int64_t bt_stride;
  int capacity;  // keys that a table row can address
  int num_blocks, block_size;
  float per_block;  // 1 / block_size
  const int32_t* q_start;
  const int32_t* q_len;
  const int32_t* t_len;
  int rows, tokens, hkv, group, window;
  int slots;          // workgroups that run at a time
  float scale_log2;   // |scale| log2 e
  uint32_t q_keep, q_sign;  // a scale of 0 clears the queries, the sign bits turn with a negative one
  PlanHeader* header;
  Part* parts;
  Part* joins;        // items of several parts
  float* pieces;
  int32_t* status;
};

// Keys of one item: [first, end), and its tiles of keys from `first` on.
struct Keys {
  int first, end, tiles;
};
__device__ __forceinline__ Keys item_keys(const ChunkArgs& a, int len, int seen, int tile) {
  const int r0 = tile * kItemRows, r1 = min(r0 + kItemRows, len * a.group) - 1;
  Keys k;
  k.end = max(seen + r1 / a.group + 1, 0);
  k.first = max(seen + r0 / a.group + 1 - a.window, 0) & ~31;
  k.tiles = ceil_div(max(k.end - k.first, 0), kTile);
  return k;
}

// ---------------------------------------------------------------------------------------------
// The plan: one workgroup.
// ---------------------------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;
static_assert(kPlanThreads == kMaxRows, "a thread a row");

__device__ __forceinline__ int plan_scan(int v, int* sums, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int inclusive = wave_inclusive_scan(v);
  if (lane == 63) sums[wave] = inclusive;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) before += sums[w];
    total += sums[w];
  }
  __syncthreads();
  return before + inclusive - v;
}

__global__ __launch_bounds__(kPlanThreads) void chunk_plan_kernel(ChunkArgs a) {
  __shared__ int sums[kPlanThreads / 64];
  __shared__ int first_item[kMaxRows + 1], row_start[kMaxRows], row_len[kMaxRows], row_seen[kMaxRows];
  __shared__ unsigned long long work;
  constexpr int kSizes = 64;  // classes of part sizes
  __shared__ int begin[kSizes + 1], slots, joins;
  const int b = threadIdx.x;
  int start = 0, len = 0, keys = 0;
  bool bad = false;
  if (b < a.rows) {
    start = a.q_start[b], len = a.q_len[b], keys = a.t_len[b];
    if (len < 0) len = 0;
    bad = len > 0 && (start < 0 || len > a.tokens || start > a.tokens - len);
    if (bad) len = 0;
    if (keys > a.capacity && a.status) {
      __hip_atomic_fetch_or(a.status, static_cast<int>(kStatusLength), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    keys = min(max(keys, 0), a.capacity);
  }
  // Rows that would bring the sum over the query's own tokens (rows that overlap) are left out, with
  // the rows behind them, which also bounds the workspace.  Sums are cut short of 32 bits: a row has
  // at most 2^20 tokens, and 1024 of them reach 2^30.
  int total = 0;
  const int at = plan_scan(len, sums, total);
  if (len > 0 && at + len > a.tokens) {
    bad = true;
    len = 0;
  }
  if (bad && a.status) {
    __hip_atomic_fetch_or(a.status, static_cast<int>(kStatusRow), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  int items = 0;
  const int item = plan_scan(ceil_div(len * a.group, kItemRows), sums, items);
  first_item[b] = item;
  row_start[b] = start, row_len[b] = len, row_seen[b] = keys - len;
  if (b == 0) first_item[kMaxRows] = items, work = 0, slots = 0, joins = 0;
  if (b <= kSizes) begin[b] = 0;
  if (b < 64) a.header->zeros[b] = 0;
  __syncthreads();
  // An item's row and its key tiles (at least one: an item without keys has an output).  A thread's first
  // item, for most calls its only one, is looked up once.
  struct Found {
    int row, tiles;
  };
  auto find = [&](int i) {
    const int r = find_row(first_item, kMaxRows, i);
    return Found{r, max(item_keys(a, row_len[r], row_seen[r], i - first_item[r]).tiles, 1)};
  };
  const Found first = b < items ? find(b) : Found{0, 0};
  auto found = [&](int i) { return i == b ? first : find(i); };
  unsigned long long mine = 0;
  for (int i = b; i < items; i += kPlanThreads) mine += found(i).tiles;
  if (mine) atomicAdd(&work, mine);
  __syncthreads();
  // A part is an equal share of the work at most, so that the last ones to run end together.  (An item has at
  // most 2^24 tiles.  The share's four roundings, of 2^-24 each, may not make it less than equal.)
  const float share = static_cast<float>(work) * static_cast<float>(a.hkv) / static_cast<float>(a.slots);
  const int cap = max(static_cast<int>(fminf(ceilf(share * (1.f + 0x1p-20f)), 0x1p25f)), kMinPart);
  const float classes = static_cast<float>(kSizes) / static_cast<float>(cap + 1);
  auto size_class = [&](int size) { return kSizes - 1 - min(static_cast<int>(static_cast<float>(size) * classes), kSizes - 1); };
  for (int i = b; i < items; i += kPlanThreads) {
    const int n = found(i).tiles, parts = ceil_div(n, cap);
    atomicAdd(&begin[size_class(n / parts) + 1], parts);
  }
  __syncthreads();
  if (b < 64) {
    static_assert(kSizes == 64, "a lane a class");
    const int inclusive = wave_inclusive_scan(begin[b + 1]);
    begin[b + 1] = inclusive;
    if (b == 63) a.header->parts = inclusive;
  }
  __syncthreads();
  for (int i = b; i < items; i += kPlanThreads) {
    const auto [r, n] = found(i);
    Part p{row_start[r], row_len[r], row_seen[r], r, i - first_item[r], 0, 0, 0};
    p.parts = ceil_div(n, cap);
    const int place = atomicAdd(&begin[size_class(n / p.parts)], p.parts);
    if (p.parts > 1) {
      p.slot = atomicAdd(&slots, p.parts);
      a.joins[atomicAdd(&joins, 1)] = p;
    }
    for (; p.part < p.parts; ++p.part) a.parts[place + p.part] = p;
  }
  __syncthreads();
  if (b == 0) a.header->joins = joins;
}

// ---------------------------------------------------------------------------------------------
// Attention.
// ---------------------------------------------------------------------------------------------
// What the loop over keys needs of the arguments, for one KV head; the rest is read again behind it, so that
// scalar registers last.
struct Cache {
  uint64_t k, v;  // of the KV head
  int64_t k_block, v_block;
  uint32_t k_token, v_token;
  int num_blocks, block_size;
  float per_block, scale_log2;
  int32_t* status;
  uint64_t zeros;
};

// (n + 0.5) / size in floating point gives the exact quotient for n < 2^22: the half keeps it away from
// the integers by 0.5 / size, more than the 2^-23 relative error of a product with a rounded reciprocal.
__device__ __forceinline__ int pages_in(const Cache& a, int n) {
  return static_cast<int>((static_cast<float>(n) + 0.5f) * a.per_block);
}

// A part's tiles of keys, one after the other.  One load of a wave takes kPerLoad neighbouring keys; a part
// begins at a multiple of 32 keys, so where the page size is a multiple of kPerLoad they lie in one page and
// the address is the wave's (WHOLE; 4096 tokens on themselves 165 us, and 304 with an address a lane).  The lanes then look up the pages of the wave's loads of many tiles
// together, a run: lane i's load is load i % kLoads of tile i / kLoads of the run.
struct Tile {
  int key, left;  // its first key, and the keys from it on to the part's end
};
struct Run {
  int page, in;  // the lane's load: its page, and the first key's place in it
};
// Places of a run in one of the caches, in the lanes, and which of the loads there is a page and a key for.
struct Places {
  uint64_t at, fine;
};

template <int D, bool WHOLE>
__device__ __forceinline__ Run look_up(const Cache& a, const int32_t* table, int wave, const Tile& x) {
  using C = Chunk<D>;
  Run r{0, 0};
  if (!WHOLE || x.left <= 0) return r;
  const int lane = fresh_thread() & 63, tile = lane / C::kLoads, i = lane % C::kLoads;
  const int t = x.key + min(tile * kTile + (wave * C::kLoads + i) * C::kPerLoad, (x.left - 1) & ~(C::kPerLoad - 1));
  const int index = t / a.block_size;
  r.in = t - index * a.block_size;
  r.page = table[index];
  return r;
}

template <int D, bool WHOLE, bool VALUES>
__device__ __forceinline__ Places find_places(const Cache& a, const Run& r, int wave, const Tile& x) {
  using C = Chunk<D>;
  Places p{0, 0};
  if (!WHOLE || x.left <= 0) return p;
  const int lane = fresh_thread() & 63, t = lane / C::kLoads * kTile + (wave * C::kLoads + lane % C::kLoads) * C::kPerLoad;
  const bool exists = static_cast<unsigned>(r.page) < static_cast<unsigned>(a.num_blocks);
  p.fine = __ballot(exists && t < x.left);
  const uint32_t page = exists ? r.page : 0, in = r.in;
  p.at = VALUES ? a.v + page * a.v_block + in * a.v_token : a.k + page * a.k_block + in * a.k_token;
  return p;
}

// Where a lane's piece of load i lies after the load's first key, in bytes.  (The turns of the pieces repeat
// every 16 keys, which a wave's loads are a multiple of apart.)
template <int D, bool VALUES>
__device__ __forceinline__ uint32_t piece_offset(const Cache& a, int lane, int i) {
  using C = Chunk<D>;
  const int piece = lane % C::kPieces, mine = lane / C::kPieces, key = (i * C::kPerLoad + mine) % 16;
  return mine * (VALUES ? a.v_token : a.k_token) +
         16 * (VALUES ? piece_at<D>(key, piece) - key * C::kPieces : piece ^ key_turn<D>(key));
}

template <int D, int I = 0>
__device__ __forceinline__ void send_whole(uint64_t place, int first, const uint32_t (&offset)[Chunk<D>::kLoads], uint32_t to) {
  using C = Chunk<D>;
  if constexpr (I < C::kLoads) {
    load_lds<I * C::kPerLoad * C::kRowBytes>(lane_value(place, first + I), offset[I], to);
    send_whole<D, I + 1>(place, first, offset, to);
  }
}

// A page a lane; zeros for loads past the part's end and for keys of a page out of range.
template <int D, bool VALUES>
__device__ __forceinline__ void send_lanes(const Cache& a, const int32_t* table, const Tile& x, int wave, uint32_t to) {
  using C = Chunk<D>;
  const int lane = fresh_thread() & 63;
#pragma unroll 1
  for (int i = 0; i < C::kLoads; ++i) {
    const int first = (wave * C::kLoads + i) * C::kPerLoad, key = first + lane / C::kPieces;
    const int n = x.key + min(key, x.left - 1), index = n / a.block_size, page = table[index];
    const uint32_t token_bytes = VALUES ? a.v_token : a.k_token, in = n - index * a.block_size;
    const bool exists = static_cast<unsigned>(page) < static_cast<unsigned>(a.num_blocks);
    if (!exists && a.status) {
      __hip_atomic_fetch_or(a.status, static_cast<int>(kStatusPage), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    const uint64_t from = (VALUES ? a.v : a.k) + page * (VALUES ? a.v_block : a.k_block) + in * token_bytes +
                          (piece_offset<D, VALUES>(a, lane, i) - lane / C::kPieces * token_bytes);
    load_lds<0>(exists && first < x.left ? from : a.zeros, uniform(to + i * C::kPerLoad * C::kRowBytes));
  }
}

// Sends the wave's part of a tile's keys (or values), tile `tile` of a run, to shared memory.
template <int D, bool WHOLE, bool VALUES>
__device__ __forceinline__ void send(const Cache& a, const int32_t* table, const Tile& x, const Places& p, int tile,
                                     const uint32_t (&offset)[Chunk<D>::kLoads], int wave, uint32_t to) {
  using C = Chunk<D>;
  if (x.left <= 0) return;
  constexpr uint32_t kAll = (1u << C::kLoads) - 1;
  if (WHOLE && (static_cast<uint32_t>(p.fine >> (tile * C::kLoads)) & kAll) == kAll) {
    send_whole<D>(p.at, tile * C::kLoads, offset, to);
  } else {
    send_lanes<D, VALUES>(a, table, x, wave, to);
  }
}

// A wave's softmax state for its 32 query rows (one per lane column): running maximum, the lane's
// part of the sum, and the unnormalised output of the lane's dimensions.
template <int D>
struct Softmax {
  f32x16 acc[Chunk<D>::kBlocks];
  float m, l;
};

// A masked key of a tile may hold infinities or NaN, which a probability of 0 does not cancel in the
// product, while another column sees that key.  In tiles with a mask such values are replaced by 0 in
// shared memory, before a barrier, each wave those that it sent; returns whether there was one.
template <int DT, int D>
__device__ __forceinline__ bool clear_not_finite(char* values, int wave) {
  using C = Chunk<D>;
  constexpr uint32_t kExponent = DT == DS_BF16 ? 0x7f80u : 0x7c00u;
  u32x4* mine = reinterpret_cast<u32x4*>(values) + wave * C::kLoads * 64 + (fresh_thread() & 63);
  bool any = false;
#pragma unroll
  for (int i = 0; i < C::kLoads; ++i) {
    u32x4 x = mine[64 * i];
    bool found = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) found |= not_finite2(x[e], kExponent);
    if (found) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] &= ((x[e] & kExponent) == kExponent ? 0u : 0xffffu) |
                ((x[e] & (kExponent << 16)) == (kExponent << 16) ? 0u : 0xffff0000u);
      }
      mine[64 * i] = x;
    }
    any |= found;
  }
  return __any(any);
}

// The values that were left out, from the cache, added to the columns that see them (where the sum is no
// longer finite whatever the weight): of `keys` keys from place `place` on, the lane column's query row sees
// key t where from <= t < from + count.
template <int DT, int D>
__device__ __forceinline__ void add_not_finite(const Cache& a, const int32_t* pages, int place, int keys, Softmax<D>& st,
                                               int from, unsigned count) {
  constexpr uint32_t kExponent = DT == DS_BF16 ? 0x7f80u : 0x7c00u;
  const int half = (fresh_thread() >> 5) & 1;
#pragma unroll 1
  for (int t = 0; t < keys; ++t) {
    const int index = pages_in(a, place + t), page = pages[index];
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.num_blocks)) continue;
    const uint64_t at = a.v + page * a.v_block + (place + t - index * a.block_size) * a.v_token + 8 * half;
    const bool sees = static_cast<unsigned>(t - from) < count;
#pragma unroll
    for (int j = 0; j < Chunk<D>::kBlocks; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32x2 v = *reinterpret_cast<const u32x2*>(at + 64 * j + 16 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint16_t x = static_cast<uint16_t>(v[e >> 1] >> (16 * (e & 1)));
          if (sees && (x & kExponent) == kExponent) st.acc[j][4 * i + e] += Elem<DT>::load(x);
        }
        __builtin_amdgcn_sched_barrier(0);  // or the conditions of all values are held at once
      }
    }
  }
}

// Scores of a tile's keys.  (Piece 2 s + half of a key is turned as piece `half` is, and 2 s
// then differs in bits of its own; the turn repeats every 16 keys.)
template <int DT, int D>
__device__ __forceinline__ void score(const char* keys, const u32x4 (&q)[Chunk<D>::kSteps], f32x16 (&sc)[kScores]) {
  using C = Chunk<D>;
  const int lane = fresh_thread() & 63, half = lane >> 5, t = lane & 31;
  const uint32_t at = t * C::kRowBytes + 16 * (half ^ key_turn<D>(t));
#pragma unroll
  for (int n = 0; n < kScores; ++n) {
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[n][i] = 0.f;
#pragma unroll
    for (int s = 0; s < C::kSteps; ++s) {
      sc[n] = mfma32<DT>(*reinterpret_cast<const u32x4*>(keys + (at ^ (32 * s)) + 32 * n * C::kRowBytes), q[s], sc[n]);
    }
  }
}

// One tile for one wave, whose scores are in `sc`; it then gets those of the
// next tile, whose products run while the weights are computed.
template <int DT, int D>
__device__ __forceinline__ void attend(const char* next_keys, const char* values, const u32x4 (&q)[Chunk<D>::kSteps],
                                       Softmax<D>& st, f32x16 (&sc)[kScores], float scale_log2) {
  using C = Chunk<D>;
  const int lane = fresh_thread() & 63, half = lane >> 5, l = lane & 15;
  float top = -INFINITY;
#pragma unroll
  for (int n = 0; n < kScores; ++n) {
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[n][i]);
  }
  // The reference of the exponents follows the maximum only when it is 2^8 behind: weights of up to 2^8
  // keep their relative precision, and most tiles leave the sums as they are.  In fp16 it stays 2^7 below
  // the maximum, so that weights lie in 2^-24 .. 2^15 of the type: those of a long tail of small
  // probabilities are then rounded relative to themselves down to 2^-21 of the largest.
  constexpr float kBelow = DT == DS_FP16 ? 7.f : 0.f;
  top = __builtin_fmaf(fmaxf(top, other_half(top)), scale_log2, -kBelow);
  if (__any(top > st.m + 8.f)) {
    const float m = fmaxf(st.m, top);
    // A factor that underflows, or is of sums of nothing yet, is taken as 2^-126 instead of 0, which is as near: an
    // infinity that is in the output already (the tile's own are, see add_not_finite) stays one.
    const float keep = fmaxf(__builtin_amdgcn_exp2f(st.m - m), 0x1p-126f);
    st.m = m;
    st.l *= keep;
#pragma unroll
    for (int j = 0; j < C::kBlocks; ++j) {
#pragma unroll
      for (int i = 0; i < 16; ++i) st.acc[j][i] *= keep;
    }
  }
  const float m = st.m == -INFINITY ? 0.f : st.m;
  f32x16 next[kScores];
  score<DT, D>(next_keys, q, next);
  u32x4 p[2 * kScores];
#pragma unroll
  for (int n = 0; n < kScores; ++n) {
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][i], scale_log2, -m));
      const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][i + 1], scale_log2, -m));
      // The product's operands are 16 bits, so the probabilities are rounded for it; the sum is of them as
      // computed, since the LSE is an fp32 output.
      st.l += x + y;
      p[2 * n + (i >> 3)][(i & 7) >> 1] = pack2<DT>(x, y);
    }
  }
  // The lane's own probabilities are the B operand: k-slot (half, e) of step s is key 16 s + 8 (e /
  // 4) + 4 half + e % 4 of the keys, and the values are read in that order.
  const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const lds_char*)values)) +
                        8 * (l & 1) + 16 * piece_at<D>(4 * half + (l >> 2), 2 * ((lane >> 4) & 1) + ((l & 3) >> 1));
#pragma unroll
  for (int s = 0; s < 2 * kScores; ++s) {
#pragma unroll
    for (int j = 0; j < C::kBlocks; ++j) {
      const u32x2 lo = read_values((base ^ (64 * j)) + 16 * s * C::kRowBytes);
      const u32x2 hi = read_values((base ^ (64 * j)) + (16 * s + 8) * C::kRowBytes);
      st.acc[j] = mfma32<DT>(u32x4{lo[0], lo[1], hi[0], hi[1]}, p[s], st.acc[j]);
    }
  }
#pragma unroll
  for (int n = 0; n < kScores; ++n) sc[n] = next[n];
}

// A wave's place in its item.
struct Rows {
  bool any;              // it has query rows
  int limit, lower;      // keys that the lane column's row sees: lower <= t < limit
  int item_from, item_to;  // keys that all rows of the item see
};

// The part's tiles of keys, `tiles` from key `key` on.  In shared memory the keys run a tile ahead of the values: while a tile is weighed, the next one's scores are computed, and the keys
// after that and the next values are on their way.
template <int DT, int D, bool WHOLE>
__device__ __forceinline__ void run_part(const Cache& a, const int32_t* table, int key, int end, int tiles, const Rows& rows,
                                         const u32x4 (&q)[Chunk<D>::kSteps], Softmax<D>& st,
                                         int wave, char* lds, int (&poison)[2][4]) {
  using C = Chunk<D>;
  const uint32_t to = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const lds_char*)lds)) +
                      wave * C::kLoads * C::kPerLoad * C::kRowBytes;
  uint32_t k_offset[C::kLoads], v_offset[C::kLoads];
#pragma unroll
  for (int i = 0; i < C::kLoads; ++i) {
    k_offset[i] = piece_offset<D, false>(a, threadIdx.x & 63, i);
    v_offset[i] = piece_offset<D, true>(a, threadIdx.x & 63, i);
  }
  // The keys' next tile and the run that it belongs to, the values' next tile (one before it) and its run, and the
  // run that the keys come to next.
  constexpr int kRun = 64 / C::kLoads;
  Tile x{key, end - key}, v = x;
  int x_tile = 0, v_tile = 0;  // of the run
  Run run = look_up<D, WHOLE>(a, table, wave, x), run_ahead = run;
  Places k_places = find_places<D, WHOLE, false>(a, run, wave, x), v_places{0, 0};
  auto send_keys = [&](int half) {
    if (x_tile == kRun) {
      run = run_ahead, x_tile = 0;
      k_places = find_places<D, WHOLE, false>(a, run, wave, x);
    }
    send<D, WHOLE, false>(a, table, x, k_places, x_tile, k_offset, wave, to + half * C::kStage);
    // The pages of the next run, half a run ahead.
    if (x_tile == kRun / 2) run_ahead = look_up<D, WHOLE>(a, table, wave, Tile{x.key + kRun / 2 * kTile, x.left - kRun / 2 * kTile});
    x.key += kTile, x.left -= kTile, ++x_tile;
  };
  // The values come to a run when the keys are one tile into it.
  auto send_values = [&](int half) {
    if (v_tile == kRun) v_tile = 0;
    if (v_tile == 0) v_places = find_places<D, WHOLE, true>(a, run, wave, v);
    send<D, WHOLE, true>(a, table, v, v_places, v_tile, v_offset, wave, to + (2 + half) * C::kStage);
    v.key += kTile, v.left -= kTile, ++v_tile;
  };
  send_keys(0);
  wait_loads();
  lds_barrier();
  send_values(0);
  send_keys(1);
  f32x16 sc[kScores];
  if (rows.any) score<DT, D>(lds, q, sc);
  const unsigned count = max(rows.limit - rows.lower, 0);
  for (int i = 0; i < tiles; ++i, key += kTile) {
    const int here = i & 1;  // the tile's half of shared memory
    wait_loads();
    char* values = lds + (2 + here) * C::kStage;
    const bool item_masked = key < rows.item_from || key + kTile > rows.item_to;
    if (item_masked) {
      const bool found = clear_not_finite<DT, D>(values, wave);
      if ((fresh_thread() & 63) == 0) poison[here][wave] = found;
    }
    lds_barrier();
    send_values(here ^ 1);
    send_keys(here);
    if (!rows.any) continue;
    if (item_masked) {
      // Also for a wave whose rows see the whole tile: the values were cleared for all waves.
      const int from = rows.lower - key, half = (fresh_thread() >> 5) & 1;
      if (__any(poison[here][fresh_thread() & 3])) {
        const int page = key / a.block_size;
        add_not_finite<DT, D>(a, table + page, key - page * a.block_size, min(kTile, end - key), st, from, count);
      }
#pragma unroll
      for (int n = 0; n < kScores; ++n) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if (static_cast<unsigned>(32 * n + 8 * (e >> 2) + (e & 3) + 4 * half - from) >= count) sc[n][e] = -INFINITY;
        }
      }
    }
    attend<DT, D>(lds + (here ^ 1) * C::kStage, values, q, st, sc, a.scale_log2);
  }
}

// A piece in the workspace: 128 maxima and 128 sums, then the outputs as the waves hold them
// ([query block][4 x dimension group][lane] of 4 floats).
template <int D>
__device__ __forceinline__ float* piece_at_slot(const ChunkArgs& a, int slot) {
  return a.pieces + static_cast<int64_t>(slot) * (kItemRows * (D + 2));
}

// Four neighbouring dimensions of one query row's result, and its LSE.
template <int DT>
__device__ __forceinline__ void store_out(const ChunkArgs& a, int token, int head, int dim, f32x4 x, float l) {
  x *= l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;  // nothing seen: zeros; NaN stays NaN
  uint16_t* out = a.out + token * a.o_row + head * a.o_head + dim;
  *reinterpret_cast<u32x2*>(out) = u32x2{pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3])};
}
__device__ __forceinline__ void store_lse(const ChunkArgs& a, int token, int head, float m, float l) {
  if (a.lse) a.lse[token * a.l_row + head * a.l_head] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2P;
}

template <int DT, int D, bool WHOLE>
__global__ __launch_bounds__(Chunk<D>::kThreads, chunk_waves(D)) void chunk_attention_kernel(ChunkArgs a) {
  using C = Chunk<D>;
  __shared__ __attribute__((aligned(512))) char lds[4 * C::kStage];
  __shared__ int poison[2][4];
  const int entry = blockIdx.x / a.hkv, h = blockIdx.x - entry * a.hkv;
  if (entry >= a.header->parts) return;
  const Part p = a.parts[entry];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), half = lane >> 5;
  const int rows = p.len * a.group;
  const int r0 = p.tile * kItemRows + 32 * wave, r = r0 + (lane & 31);
  const int token = min(r, rows - 1) / a.group, head = h * a.group + min(r, rows - 1) - token * a.group;
  Rows w;
  w.any = r0 < rows;
  w.limit = p.seen + token + 1;
  w.lower = max(w.limit - a.window, 0);
  w.item_to = p.seen + p.tile * kItemRows / a.group + 1;
  w.item_from = max(p.seen + (min((p.tile + 1) * kItemRows, rows) - 1) / a.group + 1 - a.window, 0);
  u32x4 q[C::kSteps];
  {
    const uint16_t* src = a.q + (p.start + token) * a.q_row + head * a.q_head + 8 * half;
#pragma unroll
    for (int s = 0; s < C::kSteps; ++s) q[s] = (*reinterpret_cast<const u32x4*>(src + 16 * s) & a.q_keep) ^ a.q_sign;
  }
  Softmax<D> st;
#pragma unroll
  for (int j = 0; j < C::kBlocks; ++j) {
#pragma unroll
    for (int i = 0; i < 16; ++i) st.acc[j][i] = 0.f;
  }
  st.m = -INFINITY;
  st.l = 0.f;
  const Keys keys = item_keys(a, p.len, p.seen, p.tile);
  const int first = static_cast<int>(static_cast<int64_t>(keys.tiles) * p.part / p.parts);
  const int last = static_cast<int>(static_cast<int64_t>(keys.tiles) * (p.part + 1) / p.parts);
  if (first < last) {
    const int key = keys.first + first * kTile, end = min(keys.end, keys.first + last * kTile);
    const int32_t* table = a.table + p.row * a.bt_stride;
    const Cache cache{reinterpret_cast<uint64_t>(a.k) + h * a.k_head, reinterpret_cast<uint64_t>(a.v) + h * a.v_head,
                      a.k_block, a.v_block, static_cast<uint32_t>(a.k_token), static_cast<uint32_t>(a.v_token),
                      a.num_blocks, a.block_size, a.per_block, a.scale_log2, a.status,
                      reinterpret_cast<uint64_t>(a.header->zeros)};
    run_part<DT, D, WHOLE>(cache, table, key, end, last - first, w, q, st, wave, lds, poison);
  }
  st.l += other_half(st.l);
  constexpr int kGroups = 4 * C::kBlocks;
  auto group = [&](int g) {
    return f32x4{st.acc[g >> 2][4 * (g & 3)], st.acc[g >> 2][4 * (g & 3) + 1], st.acc[g >> 2][4 * (g & 3) + 2],
                 st.acc[g >> 2][4 * (g & 3) + 3]};
  };
  if (r >= rows) return;
  const ChunkArgs z = arguments<ChunkArgs>();
  if (p.parts == 1) {
#pragma unroll
    for (int g = 0; g < kGroups; ++g) store_out<DT>(z, p.start + token, head, 8 * g + 4 * half, group(g), st.l);
    if (half == 0) store_lse(z, p.start + token, head, st.m, st.l);
    return;
  }
  float* sums = piece_at_slot<D>(z, (p.slot + p.part) * z.hkv + h);
  if (half == 0) {
    sums[32 * wave + lane] = st.m;
    sums[kItemRows + 32 * wave + lane] = st.l;
  }
  f32x4* o = reinterpret_cast<f32x4*>(sums + 2 * kItemRows) + wave * kGroups * 64 + lane;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) o[g * 64] = group(g);
}

// Joins the parts of 32 query rows of an item: a wave takes a quarter of the dimensions.
template <int DT, int D>
__global__ __launch_bounds__(256) void chunk_join_kernel(ChunkArgs a) {
  constexpr int kMine = D / 32;  // groups of four dimensions of a wave's lane
  if (static_cast<int>(blockIdx.x) >= a.header->joins) return;
  const Part p = a.joins[blockIdx.x];
  const int h = blockIdx.z, block = blockIdx.y, rows = p.len * a.group;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), half = lane >> 5;
  const int r0 = p.tile * kItemRows + 32 * block, r = r0 + (lane & 31);
  if (r >= rows) return;
  float m = -INFINITY, l = 0.f;
  f32x4 acc[kMine];
#pragma unroll
  for (int k = 0; k < kMine; ++k) acc[k] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < p.parts; ++i) {
    const float* sums = piece_at_slot<D>(a, (p.slot + i) * a.hkv + h);
    const float om = sums[32 * block + (lane & 31)], ol = sums[kItemRows + 32 * block + (lane & 31)];
    const f32x4* o = reinterpret_cast<const f32x4*>(sums + 2 * kItemRows) + (block * (D / 8) + wave * kMine) * 64 + lane;
    const float top = fmaxf(m, om);
    const float mine = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    const float other = om == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(om - top);
    m = top;
    l = l * mine + ol * other;
#pragma unroll
    for (int k = 0; k < kMine; ++k) acc[k] = acc[k] * mine + o[k * 64] * other;
  }
  const int token = r / a.group, head = h * a.group + r - token * a.group;
#pragma unroll
  for (int k = 0; k < kMine; ++k) store_out<DT>(a, p.start + token, head, 8 * (wave * kMine + k) + 4 * half, acc[k], l);
  if (wave == 0 && half == 0) store_lse(a, p.start + token, head, m, l);
}

// Bounds of a plan.  Items: whole ones and a last one a row.  A cut item has at most twice the parts that
// its tiles fill, so all cut items have at most two parts per workgroup that runs at a time, and each
// part counts once for every KV head.
struct Bounds {
  int64_t items, parts, joins, pieces;
};
Bounds plan_bounds(int rows, int tokens, int num_q_heads, int num_kv_heads, int d) {
  const int64_t group = num_q_heads / num_kv_heads;
  Bounds b;
  b.items = static_cast<int64_t>(tokens) * group / kItemRows + std::min(rows, tokens);
  const int64_t cut = 2 * static_cast<int64_t>(part_slots(d)) / num_kv_heads + 1;
  b.parts = b.items + cut;
  b.joins = std::min(b.items, cut / 2 + 1);
  b.pieces = cut * num_kv_heads;
  return b;
}
constexpr size_t kPlanHeader = sizeof(PlanHeader);
size_t rounded(size_t n) { return (n + 255) & ~size_t{255}; }

size_t chunk_workspace_bytes(int rows, int tokens, int num_q_heads, int num_kv_heads, int d) {
  if (rows <= 0 || tokens <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads) return 0;
  if (d != 64 && d != 128 && d != 256) return 0;
  const Bounds b = plan_bounds(rows, tokens, num_q_heads, num_kv_heads, d);
  return kPlanHeader + rounded((b.parts + b.joins) * sizeof(Part)) +
         static_cast<size_t>(b.pieces) * kItemRows * (d + 2) * sizeof(float);
}

template <int DT, int D>
int launch(hipStream_t stream, const ChunkArgs& a, const Bounds& b) {
  chunk_plan_kernel<<<1, kPlanThreads, 0, stream>>>(a);
  const int groups = static_cast<int>(b.parts * a.hkv);
  if (a.block_size % Chunk<D>::kPerLoad == 0) {
    chunk_attention_kernel<DT, D, true><<<groups, Chunk<D>::kThreads, 0, stream>>>(a);
  } else {
    chunk_attention_kernel<DT, D, false><<<groups, Chunk<D>::kThreads, 0, stream>>>(a);
  }
  chunk_join_kernel<DT, D><<<dim3(static_cast<int>(b.joins), kItemRows / 32, a.hkv), 256, 0, stream>>>(a);
  return check_launch("ds_chunk_attention");
}

template <int DT>
int launch_dim(hipStream_t stream, int d, const ChunkArgs& a, const Bounds& b) {
  if (d == 64) return launch<DT, 64>(stream, a, b);
  if (d == 128) return launch<DT, 128>(stream, a, b);
  return launch<DT, 256>(stream, a, b);
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int chunk_attention_impl(hipStream_t stream, const ds_chunk_attention_desc* d) {
  DS_REQUIRE(d != nullptr, "null descriptor");
  DS_REQUIRE(d->dtype == DS_BF16 || d->dtype == DS_FP16, "queries and KV caches must use BF16 or FP16");
  DS_REQUIRE(d->rows >= 0 && d->tokens >= 0, "row and token counts must be non-negative");
  DS_REQUIRE(d->num_q_heads > 0 && d->num_kv_heads > 0 && d->num_q_heads % d->num_kv_heads == 0,
             "query heads must be divisible by KV heads");
  DS_SUPPORTED(d->head_dim == 64 || d->head_dim == 128 || d->head_dim == 256, "head_dim must be 64, 128 or 256");
  DS_SUPPORTED(d->rows <= kMaxRows, "at most %d rows", kMaxRows);
  DS_REQUIRE(d->block_size > 0 && d->num_blocks > 0 && d->max_blocks > 0, "block sizes and counts must be positive");
  DS_REQUIRE(d->window >= 0, "window must not be negative (0: no window)");
  DS_SUPPORTED(d->block_size <= (1 << 20), "at most 2^20 tokens per page");
  if (d->rows == 0 || d->tokens == 0) return clear_error();
  DS_REQUIRE(d->query && d->output && d->key_cache && d->value_cache && d->block_table && d->query_start &&
                 d->query_len && d->target_len,
             "null tensor pointer");
  const int64_t strides[] = {d->q_row_stride,   d->q_head_stride,  d->o_row_stride,   d->o_head_stride, d->k_block_stride,
                             d->k_token_stride, d->k_head_stride,  d->v_block_stride, d->v_token_stride, d->v_head_stride};
  for (int64_t s : strides) DS_REQUIRE(s >= 0 && s % 8 == 0, "row, page and head strides must be multiples of 8 elements");
  // Places within a page are 32-bit byte counts.
  for (int i = 4; i < 10; ++i) DS_SUPPORTED(strides[i] < (1 << 30), "pages of at most 2^30 elements");
  DS_SUPPORTED(d->block_size * d->k_token_stride + d->num_kv_heads * d->k_head_stride < (1 << 30) &&
                   d->block_size * d->v_token_stride + d->num_kv_heads * d->v_head_stride < (1 << 30),
               "pages of at most 2^30 elements");
  DS_REQUIRE(aligned(d->query) && aligned(d->output) && aligned(d->key_cache) && aligned(d->value_cache),
             "query, output and KV caches must be 16-byte aligned");
  const size_t need = chunk_workspace_bytes(d->rows, d->tokens, d->num_q_heads, d->num_kv_heads, d->head_dim);
  DS_REQUIRE(d->workspace && d->workspace_bytes >= need && (reinterpret_cast<uintptr_t>(d->workspace) & 255u) == 0,
             "workspace must be 256-byte aligned and hold ds_chunk_attention_workspace_bytes()");
  const int group = d->num_q_heads / d->num_kv_heads;
  const Bounds b = plan_bounds(d->rows, d->tokens, d->num_q_heads, d->num_kv_heads, d->head_dim);
  DS_SUPPORTED(d->tokens <= (1 << 20), "at most 2^20 query tokens");
  DS_SUPPORTED(static_cast<int64_t>(d->tokens) * group < (1 << 30) && d->num_kv_heads <= 65535 &&
                   b.parts * d->num_kv_heads < (1 << 24),
               "too many query tokens or heads for one launch");
  ChunkArgs a{};
  a.q = static_cast<const uint16_t*>(d->query);
  a.q_row = d->q_row_stride, a.q_head = d->q_head_stride;
  a.out = static_cast<uint16_t*>(d->output);
  a.o_row = d->o_row_stride, a.o_head = d->o_head_stride;
  a.lse = d->lse;
  a.l_row = d->lse_token_stride, a.l_head = d->lse_head_stride;
  a.k = static_cast<const char*>(d->key_cache);
  a.k_block = 2 * d->k_block_stride, a.k_token = 2 * d->k_token_stride, a.k_head = 2 * d->k_head_stride;
  a.v = static_cast<const char*>(d->value_cache);
  a.v_block = 2 * d->v_block_stride, a.v_token = 2 * d->v_token_stride, a.v_head = 2 * d->v_head_stride;
  a.table = d->block_table;
  a.bt_stride = d->bt_stride;
  a.capacity = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(d->max_blocks) * d->block_size, 1 << 30));
  a.num_blocks = d->num_blocks;
  a.block_size = d->block_size;
  a.per_block = 1.f / static_cast<float>(d->block_size);
  a.q_start = d->query_start, a.q_len = d->query_len, a.t_len = d->target_len;
  a.rows = d->rows, a.tokens = d->tokens, a.hkv = d->num_kv_heads, a.group = group;
  a.window = d->window ? std::min(d->window, 1 << 30) : 1 << 30;  // rows have at most 2^30 keys
  a.slots = part_slots(d->head_dim);
  // Masked scores are -infinity, which a scale of 0 must not meet.
  a.scale_log2 = d->scale == 0.f ? 1.f : std::fabs(d->scale) * kLog2eP;
  a.q_keep = d->scale == 0.f ? 0u : ~0u;
  a.q_sign = d->scale < 0.f ? 0x80008000u : 0u;
  char* work = static_cast<char*>(d->workspace);
  a.header = reinterpret_cast<PlanHeader*>(work);
  a.parts = reinterpret_cast<Part*>(work + kPlanHeader);
  a.joins = a.parts + b.parts;
  a.pieces = reinterpret_cast<float*>(work + kPlanHeader + rounded((b.parts + b.joins) * sizeof(Part)));
  a.status = d->status;
  return d->dtype == DS_BF16 ? launch_dim<DS_BF16>(stream, d->head_dim, a, b)
                             : launch_dim<DS_FP16>(stream, d->head_dim, a, b);
}

}  // namespace
}  // namespace ds355

extern "C" size_t ds_chunk_attention_workspace_bytes(int rows, int tokens, int num_q_heads, int num_kv_heads,
                                                     int head_dim) {
  return ds355::chunk_workspace_bytes(rows, tokens, num_q_heads, num_kv_heads, head_dim);
}

extern "C" int ds_chunk_attention(ds_stream_t stream, const ds_chunk_attention_desc* desc) {
  return ds355::chunk_attention_impl(reinterpret_cast<hipStream_t>(stream), desc);
}

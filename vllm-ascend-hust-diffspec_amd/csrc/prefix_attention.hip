// Paged attention of a verified batch that shares a long prefix, computed once for all rows.
//
// The verifier's side of a step: ragged rows of query tokens (query_start, query_len) attend over
// their paged keys and values (block_table, target_len), causally at the end, and the natural-log
// LSE of every query head comes back with the output: the snapshot the chunk scoring takes
// (diffspec/runtime.py:841-878 captures both from the target's fused attention).  All rows agree on
// their first prefix_len tokens.
//
//   L(b, i) = target_len[b] - query_len[b] + i + 1         keys that query token i of row b sees
//   out     = sum_{t < L} softmax_t(scale q . k_t) v_t,  lse = ln sum_{t < L} exp(scale q . k_t)
//
// The prefix is one problem for the whole batch: the query heads of all rows' tokens that share a
// KV head are rows of one matrix, so every prefix key is read once per 128 (or 64) of them instead
// of once per request.  Each row's own tokens (prefix_len .. target_len) are a problem of the row.
// Softmax pieces over disjoint key ranges join exactly: with m the maximum, l the sum of
// exp(x - m) and O the sum of exp(x - m) v of each piece, out = sum_i 2^(m_i - m) O_i / sum_i
// 2^(m_i - m) l_i (base 2 here, the logits pre-scaled by log2 e).
//
// Work: a unit is (KV head, tile of query rows, key range); its key tiles are laid end to end with
// all other units' and dealt to the workgroups in equal contiguous shares, whatever the rows'
// lengths (a unit also counts a few places for what it costs beside its tiles).  Every workgroup
// derives the same layout from the lengths on the device, so a captured launch follows changed
// lengths.  Prefix ranges are cut into segments of one share with the row
// tiles inside a segment next to each other, and consecutive shares are given to one XCD, so the
// row tiles that read the same keys do it at about the same time behind one L2.  A share that ends
// inside a unit leaves its piece (m, l, O in fp32) in the workspace; prefix_join_kernel joins them.
//
// Measured (32 query heads on 4, 128 dimensions, bf16; this kernel + the join, back to back): 16 rows of 5
// tokens over 32 k shared keys and up to 4 k of their own 89 us (46 GFLOP: 517 TFLOP/s; a large library product
// reaches 1157): no unit is saturated (of the CUs' busy cycles the matrix units take 28%, vector issue 44%,
// shared memory 32%), waves wait for 37% of theirs, and a SIMD's two waves meet at every tile's barrier, so that
// products, softmax and staging add up; one token each over 16 k 39 us (2.3 TB/s; a large copy reaches 5.1), bound by
// loads' latency and the units' ends; two rows over 1 k 15 us, two launches' latency.  A prompt chunk that
// attends mostly to itself takes about three times its products (4096 tokens, 32 heads on 8: 416 us, floor
// 119): all query tiles of a row count as many key tiles as the last, and those past a tile's own end are
// staged as zeros.
#include <cmath>

#include "ds355_common.h"

namespace ds355 {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float kLog2eP = 1.44269504088896340736f;
constexpr float kLn2P = 0.69314718055994530942f;
constexpr int kWideRows = 128, kNarrowRows = 64;  // query rows of a unit's tile
constexpr uint32_t kStatusRow = 1;     // a row's query tokens are out of range
constexpr uint32_t kStatusLength = 2;  // a row is longer than its block table
constexpr uint32_t kStatusPage = 4;    // a page id is out of range

// Keys per tile: 32 KiB of keys and of values, 16 of each for 256 dimensions.
constexpr int tile_keys(int d) { return d <= 128 ? 16384 / d : 8192 / d; }
// Places that a unit takes in the work beside its key tiles: what its queries' loads, its joins and its
// piece cost, in tiles.  Measured in us: for 128 dimensions, 80 query tokens over 32 k shared keys 99 (1),
// 91 (2 to 4), 92 (6); for 64, 57 ragged rows over 5 k 85.5 (1), 75.8 (2), 74.8 (3), 81.5 (4), 87.1 (6);
// for 256, 80 tokens over 16 k 75 (2), 70 (3), 64 (5), 62 (8), and 48 rows over 4 k 104, 102, 100, 106.
constexpr int unit_cost(int d) { return d <= 128 ? 3 : 5; }

template <int D>
struct Shape {
  // A wave holds its queries and outputs in registers, which 256 dimensions do not fit: there two waves
  // take half of the dimensions each of 32 query rows, and add up their parts of the scores through shared
  // memory.  48 rows of two tokens, 32 heads on 8, over 4 k shared keys and 100 to 900 of their own: 102 us;
  // with four waves of twice the registers, which spilled some between the tiles, 232.
  static constexpr int kHalves = D <= 128 ? 1 : 2;
  static constexpr int kWaves = 8;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kTile = tile_keys(D);
  static constexpr int kUnitCost = unit_cost(D);
  static constexpr int kLanes = D / 8;                // 16-byte pieces of a key
  static constexpr int kPerPass = kThreads / kLanes;  // keys that one load of all threads covers
  static constexpr int kPerLoad = 64 / kLanes;        // keys that one load of a wave covers
  static constexpr int kPasses = kTile / kPerPass;
  // A staged key takes 16 bytes more than its elements, so that the 16-byte reads of eight
  // neighbouring keys touch different banks; values lie close, their pieces turned (piece_at).
  static constexpr int kKeyBytes = 2 * D + 16;
  static constexpr int kValuesAt = kTile * kKeyBytes;
  static constexpr int kStage = kValuesAt + kTile * 2 * D;  // bytes of a staged tile
  static constexpr int kSteps = D / 16 / kHalves;     // score MFMAs of a wave per 32 keys
  static constexpr int kBlocks = D / 32 / kHalves;    // its output blocks of 32 dimensions
  static constexpr int kScores = kHalves == 1 ? 0 : 4096 * kWaves;  // bytes in which the halves' scores meet
};

struct PrefixArgs {
  const uint16_t* q;
  int64_t q_row, q_head;
  uint16_t* out;
  int64_t o_row, o_head;
  float* lse;
  int64_t l_row, l_head;
  const char* k;
  uint32_t k_block, k_token, k_head;  // bytes
  const char* v;
  uint32_t v_block, v_token, v_head;
  const int32_t* table;
  int64_t bt_stride;
  int capacity;  // keys that a table row can address
  int num_blocks, block_size;
  float per_block;  // 1 / block_size
  const int32_t* q_start;
  const int32_t* q_len;
  const int32_t* t_len;
  const int32_t* prefix_len;
  int rows, tokens, hkv, group;
  float scale_log2;  // |scale| log2 e
  uint32_t q_sign;   // sign bits that a negative scale turns in the queries
  float* pieces;
  int slots;
  int groups;  // workgroups of the attention kernel
  int32_t* status;
};

// ---------------------------------------------------------------------------------------------
// The layout of the work, derived by every workgroup from the lengths.
// ---------------------------------------------------------------------------------------------
struct Plan {
  int prefix;      // shared keys
  int prefix_row;  // row whose table the prefix is read through
  int seen_by_all;  // keys that every query token sees
  int query_tokens;
  int prefix_tile;   // query rows of a prefix tile
  int row_tiles;     // prefix tiles of query rows, per KV head
  int key_tiles;     // tiles of prefix keys
  int segments, segment;  // pieces of the prefix, and the key tiles of one
  int prefix_work;   // places of all prefix units
  int prefix_units;
  int work;          // places of all units
  int share;         // places per workgroup
};

struct RowTables {
  int token[kMaxRows + 1];  // query tokens of the rows before
  int work[kMaxRows + 1];   // places of the own units of the rows before, per KV head
  int start[kMaxRows];      // first query token
  int seen[kMaxRows];       // keys that its first query token sees, less one
};

struct Row {
  int start, len, keys;
};

// Row b's query tokens and keys; len 0 for a row without query tokens or with tokens out of range.
__device__ __forceinline__ Row row_of(const PrefixArgs& a, int b) {
  Row r{a.q_start[b], a.q_len[b], a.t_len[b]};
  if (r.len <= 0 || r.start < 0 || r.len > a.tokens || r.start > a.tokens - r.len) r.len = 0;
  r.keys = min(max(r.keys, 0), a.capacity);
  return r;
}

template <int D>
__device__ __forceinline__ int tile_rows(int rows) {
  return rows > kNarrowRows || Shape<D>::kHalves == 2 ? kWideRows : kNarrowRows;
}
__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }
template <int D>
__device__ __forceinline__ int query_tiles(int rows) { return ceil_div(rows, tile_rows<D>(rows)); }

// The thread's index, opaque to the compiler: what a part of the loop derives from it is derived there
// again, instead of being kept in registers that the loop needs (spilled ones would be loaded in order
// behind the keys in flight).
__device__ __forceinline__ int fresh_thread() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// A value that is the same in all lanes, to the scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ int wave_min(int v) {
  return static_cast<int>(wave_pick<false>(static_cast<uint32_t>(v) ^ 0x80000000u) ^ 0x80000000u);
}

// What one wave's rows add to the plan, and the sums over the waves before it.
struct Part {
  int tokens, first, least, seen, cut, count;
};

// Rows are held a lane each, round by round of THREADS rows, and every wave sums the parts of all
// waves itself: one barrier for the query tokens, one for the own work, one before the tables are read.
template <int D, int THREADS>
__device__ __forceinline__ Plan make_plan(const PrefixArgs& a, RowTables& t, bool report) {
  constexpr int kTile = Shape<D>::kTile, kRounds = kMaxRows / THREADS, kParts = kMaxRows / 64;
  __shared__ Part parts[kParts];
  __shared__ int part_work[kParts];
  Plan p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int used = ceil_div(a.rows, 64);
  Row row[kRounds];
  int before[kRounds];  // query tokens before the row, of its part
  const int asked = a.prefix_len[0];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int part = i * (THREADS / 64) + wave, b = 64 * part + lane;
    row[i] = Row{0, 0, 0};
    before[i] = 0;
    if (part >= used) continue;
    if (b < a.rows) row[i] = row_of(a, b);
    const int sum = wave_inclusive_scan(row[i].len);
    before[i] = sum - row[i].len;
    const bool keys = row[i].len > 0 && row[i].keys > 0;
    const int first = wave_min(keys ? b : INT_MAX), least = wave_min(keys ? row[i].keys : INT_MAX);
    const int seen = wave_min(row[i].len > 0 ? row[i].keys - row[i].len + 1 : INT_MAX);
    const int count = __builtin_popcountll(__ballot(keys));
    if (lane == 63) parts[part] = Part{sum, first, least, seen, 0, count};
  }
  __syncthreads();
  // Rows that would bring the sum over the query's own tokens (rows that overlap) are left out, which
  // also bounds the workspace: `cut` is the sum before the first of them.
  int sum = 0, least = INT_MAX, count = 0, mine[kRounds];
  p.prefix_row = INT_MAX;
  p.seen_by_all = INT_MAX;
  for (int w = 0; w < used; ++w) {
    const Part q = parts[w];
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      if (w == i * (THREADS / 64) + wave) mine[i] = sum;
    }
    sum = min(sum + q.tokens, a.tokens + 1);
    p.prefix_row = min(p.prefix_row, q.first);
    least = min(least, q.least);
    p.seen_by_all = min(p.seen_by_all, q.seen);
    count += q.count;
  }
  const bool overlap = sum > a.tokens;
  int cut = sum;
  if (overlap) {  // the parts again, now knowing where each begins
    cut = INT_MAX;
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int part = i * (THREADS / 64) + wave;
      if (part >= used) continue;
      const int at = mine[i] + before[i];
      const int c = wave_min(at > a.tokens - row[i].len ? at : INT_MAX);
      if (lane == 63) parts[part].cut = c;
    }
    __syncthreads();
    for (int w = 0; w < used; ++w) cut = min(cut, parts[w].cut);
    cut = min(cut, a.tokens);
    __syncthreads();
  }
  // A single row has nobody to share with: all its keys are its own.
  // Key ranges begin at multiples of 16: what is left of the prefix is read row by row.
  p.prefix = count > 1 ? min(max(asked, 0), least) & ~15 : 0;
  p.prefix = uniform(p.prefix);
  p.prefix_row = uniform(count > 0 ? p.prefix_row : 0);
  p.seen_by_all = uniform(p.seen_by_all);
  p.query_tokens = uniform(cut);
  const int m = p.query_tokens * a.group;
  p.prefix_tile = tile_rows<D>(m);
  p.row_tiles = ceil_div(m, p.prefix_tile);
  p.key_tiles = ceil_div(p.prefix, kTile);
  // Own units.
  int own_work[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int part = i * (THREADS / 64) + wave, b = 64 * part + lane;
    own_work[i] = 0;
    if (part >= used) continue;
    const int at = mine[i] + before[i];
    const bool fits = at <= a.tokens - row[i].len && at + row[i].len <= cut;
    if (report && b < a.rows && a.status) {
      const uint32_t bits = ((a.q_len[b] > 0 && (row[i].len == 0 || !fits)) ? kStatusRow : 0u) |
                            (a.t_len[b] > a.capacity ? kStatusLength : 0u);
      if (bits) __hip_atomic_fetch_or(a.status, static_cast<int>(bits), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    int w = 0;
    if (row[i].len > 0 && fits && row[i].keys > p.prefix) {
      w = query_tiles<D>(row[i].len * a.group) * (Shape<D>::kUnitCost + ceil_div(row[i].keys - p.prefix, kTile));
    }
    const int work = wave_inclusive_scan(w);
    own_work[i] = work - w;
    if (lane == 63) part_work[part] = work;
    if (b < a.rows) {
      t.token[b] = min(at, cut);
      t.start[b] = row[i].start;
      t.seen[b] = row[i].keys - row[i].len;
    }
  }
  __syncthreads();
  int work = 0;
  for (int w = 0; w < used; ++w) {
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      if (w == i * (THREADS / 64) + wave) own_work[i] += work;
    }
    work += uniform(part_work[w]);
  }
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int b = 64 * (i * (THREADS / 64) + wave) + lane;
    if (b < a.rows) t.work[b] = own_work[i];
  }
  if (threadIdx.x == 0) {
    t.token[a.rows] = cut;
    t.work[a.rows] = work;
  }
  __syncthreads();
  // A segment of the prefix is a share without the cost of a unit, so that a unit is about a share.  It
  // ends at the prefix: its places times all row tiles, by which a unit is found, are then no more than
  // the work, which the host bounds.
  p.segment = min(ceil_div(a.hkv * p.row_tiles * p.key_tiles + a.hkv * work, a.groups), p.key_tiles);
  p.segment = max(1, p.segment);
  p.segments = ceil_div(p.key_tiles, p.segment);
  p.prefix_units = a.hkv * p.segments * p.row_tiles;
  p.prefix_work = a.hkv * p.row_tiles * p.key_tiles + Shape<D>::kUnitCost * p.prefix_units;
  p.work = p.prefix_work + a.hkv * work;
  p.share = max(1, ceil_div(p.work, a.groups));
  return p;
}

// One unit and where it lies in the work: kUnitCost places, then one for each of its key tiles.
struct Unit {
  int index;       // in the order of the work
  int kv_head;
  int row;         // own units: the row; prefix units: -1
  int tile;        // tile of query rows
  int rows;        // query rows in all (of the row, or of the batch)
  int tile_rows;
  int first_tile;  // place of its first key tile
  int key_tiles;
  int key0;        // first key
  int key_end;     // one past the last key
  int seen_by_all; // keys that all its query rows see
};

template <int D>
__device__ __forceinline__ Unit prefix_unit(const PrefixArgs& a, const Plan& p, int h, int segment, int tile) {
  constexpr int kTile = Shape<D>::kTile;
  Unit u;
  const int before = segment * p.segment;
  u.key_tiles = min(p.segment, p.key_tiles - before);
  u.index = (segment * a.hkv + h) * p.row_tiles + tile;
  u.kv_head = h;
  u.row = -1;
  u.tile = tile;
  u.rows = p.query_tokens * a.group;
  u.tile_rows = p.prefix_tile;
  u.first_tile = before * a.hkv * p.row_tiles + (h * p.row_tiles + tile) * u.key_tiles +
                 Shape<D>::kUnitCost * (u.index + 1);
  u.key0 = before * kTile;
  u.key_end = min(p.prefix, u.key0 + u.key_tiles * kTile);
  u.seen_by_all = min(p.seen_by_all, u.key_end);
  return u;
}

template <int D>
__device__ __forceinline__ Unit own_unit(const PrefixArgs& a, const Plan& p, const RowTables& t, int b, int h,
                                         int tile) {
  Unit u;
  const int w = t.work[b + 1] - t.work[b];
  u.rows = (t.token[b + 1] - t.token[b]) * a.group;
  const int n = query_tiles<D>(u.rows);
  // Indexes of a row's units start past those of the rows before: they have at most one tile each
  // more than whole tiles of kNarrowRows query rows.
  u.index = p.prefix_units + a.hkv * (b + t.token[b] * a.group / kNarrowRows) + h * n + tile;
  u.kv_head = h;
  u.row = b;
  u.tile = tile;
  u.tile_rows = tile_rows<D>(u.rows);
  u.key_tiles = w / n - Shape<D>::kUnitCost;
  u.first_tile = p.prefix_work + a.hkv * t.work[b] + h * w + tile * (w / n) + Shape<D>::kUnitCost;
  u.key0 = p.prefix;
  // The tile's last query token sees most.
  u.key_end = t.seen[b] + (min((tile + 1) * u.tile_rows, u.rows) - 1) / a.group + 1;
  u.seen_by_all = min(t.seen[b] + tile * u.tile_rows / a.group + 1, u.key_end);
  return u;
}

// The unit that holds place `w` of the work (the same for all lanes).
template <int D>
__device__ __forceinline__ Unit unit_at(const PrefixArgs& a, const Plan& plan, const RowTables& t, int w) {
  Plan p;
  p.prefix = uniform(plan.prefix), p.seen_by_all = uniform(plan.seen_by_all);
  p.query_tokens = uniform(plan.query_tokens), p.prefix_tile = uniform(plan.prefix_tile);
  p.row_tiles = uniform(plan.row_tiles), p.key_tiles = uniform(plan.key_tiles), p.segment = uniform(plan.segment);
  p.prefix_work = uniform(plan.prefix_work), p.prefix_units = uniform(plan.prefix_units);
  Unit u;
  if (w < p.prefix_work) {
    const int per_segment = (p.segment + Shape<D>::kUnitCost) * a.hkv * p.row_tiles;
    const int segment = w / per_segment, len = min(p.segment, p.key_tiles - segment * p.segment) + Shape<D>::kUnitCost;
    const int i = (w - segment * per_segment) / len;
    u = prefix_unit<D>(a, p, i / p.row_tiles, segment, i % p.row_tiles);
  } else {
    const int rest = w - p.prefix_work;
    int lo = 0, hi = a.rows - 1;  // the last row whose work starts at or before `rest`
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.hkv * uniform(t.work[mid]) <= rest) lo = mid; else hi = mid - 1;
    }
    const int before = uniform(t.work[lo]), mine = uniform(t.work[lo + 1]) - before;
    const int in_row = rest - a.hkv * before, h = in_row / mine;
    const int n = query_tiles<D>((uniform(t.token[lo + 1]) - uniform(t.token[lo])) * a.group);
    u = own_unit<D>(a, p, t, lo, h, (in_row - h * mine) / (mine / n));
  }
  u.index = uniform(u.index), u.kv_head = uniform(u.kv_head), u.row = uniform(u.row), u.tile = uniform(u.tile);
  u.rows = uniform(u.rows), u.tile_rows = uniform(u.tile_rows), u.first_tile = uniform(u.first_tile);
  u.key_tiles = uniform(u.key_tiles), u.key0 = uniform(u.key0), u.key_end = uniform(u.key_end);
  u.seen_by_all = uniform(u.seen_by_all);
  return u;
}

// Row of the batch that holds query token `token` of the packed order.
__device__ __forceinline__ int row_at(const PrefixArgs& a, const RowTables& t, int token) {
  int lo = 0, hi = a.rows - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.token[mid] <= token) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// A query row of a unit: its token in the query tensor, its head and the keys it sees.
struct QueryRow {
  int token, head, limit;
  bool valid;
};
__device__ __forceinline__ QueryRow query_row(const PrefixArgs& a, const RowTables& t, const Unit& u, int r) {
  QueryRow q{0, 0, INT_MAX, r < u.rows};
  if (q.valid) {
    const int token = r / a.group;
    int b = u.row, i = token;
    if (b < 0) {
      b = row_at(a, t, token);
      i = token - t.token[b];
    }
    q.token = t.start[b] + i;
    q.head = u.kv_head * a.group + (r - token * a.group);
    q.limit = t.seen[b] + i + 1;
  }
  return q;
}

// ---------------------------------------------------------------------------------------------
// Matrix products: 32x32x16, A rows and B columns of 32, k-slot (lane / 32, e) = 8 (lane / 32) + e;
// result i of a lane is row 8 (i / 4) + 4 (lane / 32) + i % 4 of column lane % 32.
// ---------------------------------------------------------------------------------------------
template <int DT>
__device__ __forceinline__ f32x16 mfma32(u32x4 x, u32x4 y, f32x16 c) {
  if constexpr (DT == DS_BF16) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0,
                                                   0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0,
                                                  0);
  }
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  if constexpr (DT == DS_BF16) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 v = {static_cast<__bf16>(x), static_cast<__bf16>(y)};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 v = {static_cast<_Float16>(x), static_cast<_Float16>(y)};
    return __builtin_bit_cast(uint32_t, v);
  }
}

// Combines a lane's value with lane ^ 32's.
__device__ __forceinline__ float other_half(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// Where 16-byte piece `c` of staged value `t` lies (in pieces): the pieces of eight neighbouring keys
// are turned against each other by two, so that a transposing read (two pieces of four keys) touches
// different banks.
template <int D>
__device__ __forceinline__ int piece_at(int t, int c) {
  const int turn = D >= 128 ? 2 * (t & 7) : 2 * ((t >> 1) & 3);
  return t * (D / 8) + (c ^ turn);
}

// (n + 0.5) / size in floating point gives the exact quotient for n < 2^22: the half keeps it away from
// the integers by 0.5 / size, more than the 2^-23 relative error of a product with a rounded reciprocal.
__device__ __forceinline__ int pages_in(const PrefixArgs& a, int n) {
  return static_cast<int>((static_cast<float>(n) + 0.5f) * a.per_block);
}

// A key tile of the share: its keys [key, key_end) and the page and place of the first one, which the
// places of the others follow by small distances.
struct Step {
  int key, key_end, head;
  const int32_t* pages;  // the table entry of the first key's page
  int place;
};

// The share's key tiles in order, across its units.
template <int D>
struct Feed {
  Unit unit;
  int at, end;  // places: the next one, the share's end
  Step step;    // of the next key tile of the unit

  __device__ __forceinline__ void start(const PrefixArgs& a, const Plan& p, const RowTables& t) {
    unit = unit_at<D>(a, p, t, at);
    at = max(at, unit.first_tile);
    step.key = unit.key0 + (at - unit.first_tile) * Shape<D>::kTile;
    step.key_end = unit.key_end;
    step.head = unit.kv_head;
    const int page = uniform(step.key / a.block_size);
    step.place = step.key - page * a.block_size;
    step.pages = a.table + static_cast<int64_t>(unit.row < 0 ? uniform(p.prefix_row) : unit.row) * a.bt_stride + page;
  }
  // The next key tile; one without keys behind the last.
  __device__ __forceinline__ Step next(const PrefixArgs& a, const Plan& p, const RowTables& t) {
    Step s = step;
    if (at >= end) {
      s.key = s.key_end = 0;
      return s;
    }
    if (++at == unit.first_tile + unit.key_tiles) {
      if (at < end) start(a, p, t);
    } else {
      const int n = uniform(pages_in(a, step.place + Shape<D>::kTile));
      step.key += Shape<D>::kTile;
      step.pages += n;
      step.place += Shape<D>::kTile - n * a.block_size;
    }
    return s;
  }
};

// A tile's keys and values in flight to shared memory.  One load of a wave takes kPerLoad neighbouring
// keys (whole 128-byte lines of one head); ranges begin at multiples of 16 keys, so where the page
// size is a multiple of kPerLoad they lie in one page and the addresses are the wave's (WHOLE).  Lane i
// of a wave looks up the page of its load i a tile ahead, and computes its place in the caches.
template <int D>
struct Staged {
  u32x4 k[Shape<D>::kPasses], v[Shape<D>::kPasses];
  int page, in;  // of the next tile's loads
  int bad;       // loads in flight whose page is out of range
};

// Loads past the range take its last keys (and are zeroed on their way to shared memory).
template <int D, bool WHOLE>
__device__ __forceinline__ void find_pages(const PrefixArgs& a, const Step& step, int wave, Staged<D>& s) {
  using S = Shape<D>;
  if (step.key >= step.key_end || !WHOLE) return;
  const int i = fresh_thread() % S::kPasses;
  const int last = (step.key_end - 1 - step.key) & ~(S::kPerLoad - 1);
  const int n = step.place + min(i * S::kPerPass + wave * S::kPerLoad, last);
  const int j = pages_in(a, n);
  s.in = n - j * a.block_size;
  s.page = step.pages[j];
}

// The places of lane i's load in the caches, in bytes.
struct Places {
  uint64_t k, v;
};
template <int D>
__device__ __forceinline__ Places load_places(const PrefixArgs& a, const Step& step, Staged<D>& s) {
  const bool fine = static_cast<unsigned>(s.page) < static_cast<unsigned>(a.num_blocks);
  s.bad = static_cast<int>(__ballot(!fine)) & ((1 << Shape<D>::kPasses) - 1);
  const uint32_t page = fine ? s.page : 0, in = s.in;
  return Places{static_cast<uint64_t>(page) * a.k_block + (in * a.k_token + step.head * a.k_head),
                static_cast<uint64_t>(page) * a.v_block + (in * a.v_token + step.head * a.v_head)};
}
__device__ __forceinline__ uint64_t place_of(uint64_t places, int i) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(places), i);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(places >> 32), i);
  return static_cast<uint64_t>(hi) << 32 | lo;
}

__device__ __forceinline__ u32x4 load_piece(const char* base, uint32_t bytes) {
  return *reinterpret_cast<const u32x4*>(base + bytes);
}

template <int D, bool WHOLE>
__device__ __forceinline__ void load_keys(const PrefixArgs& a, const Step& step, const Places& at, int thread, int wave,
                                          int i, Staged<D>& s) {
  using S = Shape<D>;
  if (step.key >= step.key_end) return;
  const int lane = thread & 63;
  const uint32_t piece = 16 * (lane % S::kLanes), mine = lane / S::kLanes;
  if constexpr (WHOLE) {
    s.k[i] = load_piece(a.k + place_of(at.k, i), mine * a.k_token + piece);
    s.v[i] = load_piece(a.v + place_of(at.v, i), mine * a.v_token + piece);
  } else {  // a page a lane
    const int key = i * S::kPerPass + wave * S::kPerLoad + static_cast<int>(mine);
    const int n = step.place + min(key, step.key_end - 1 - step.key);
    const int j = pages_in(a, n), found = step.pages[j];
    const uint32_t in = n - j * a.block_size;
    const bool fine = static_cast<unsigned>(found) < static_cast<unsigned>(a.num_blocks);
    const uint64_t page = fine ? found : 0;
    s.bad = (s.bad & ~(1 << i)) | (fine ? 0 : 1 << i);
    s.k[i] = load_piece(a.k + page * a.k_block, in * a.k_token + step.head * a.k_head + piece);
    s.v[i] = load_piece(a.v + page * a.v_block, in * a.v_token + step.head * a.v_head + piece);
  }
}

__device__ __forceinline__ bool not_finite2(uint32_t w, uint32_t exponent) {
  return (w & exponent) == exponent || (w & (exponent << 16)) == (exponent << 16);
}

// Load i's keys to shared memory, zeros for those past the range or of a page out of it (`tail`: there may
// be such).  Returns whether a value is not finite (CHECK).
template <int DT, int D, bool CHECK>
__device__ __forceinline__ bool store_keys(const PrefixArgs& a, char* stage, const Step& step, bool tail, int thread,
                                           int wave, int i, Staged<D>& s) {
  using S = Shape<D>;
  constexpr uint32_t kExponent = DT == DS_BF16 ? 0x7f80u : 0x7c00u;
  const int lane = thread & 63, piece = lane % S::kLanes;
  const int t = i * S::kPerPass + wave * S::kPerLoad + lane / S::kLanes;
  if (tail) {
    if (step.key + t >= step.key_end || (s.bad >> i) & 1) {
      s.k[i] = u32x4{0, 0, 0, 0};
      s.v[i] = u32x4{0, 0, 0, 0};
      if (step.key + t < step.key_end && a.status) {
        __hip_atomic_fetch_or(a.status, static_cast<int>(kStatusPage), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
  }
  *reinterpret_cast<u32x4*>(stage + t * S::kKeyBytes + 16 * piece) = s.k[i];
  reinterpret_cast<u32x4*>(stage + S::kValuesAt)[piece_at<D>(t, piece)] = s.v[i];
  if constexpr (!CHECK) return false;
  return not_finite2(s.v[i][0], kExponent) || not_finite2(s.v[i][1], kExponent) || not_finite2(s.v[i][2], kExponent) ||
         not_finite2(s.v[i][3], kExponent);
}

// Where a lane reads in a staged tile, in bytes: a key's piece 0 for the score product (key lane % 32
// of 32, the first 16 bytes of its half of a step), and for the output product the values of four keys
// of output block 0.  A transposing read gives lane l of 16 four keys of dimension l, where lane l names
// key l / 4 and dimensions 4 (l % 4) .. + 3; keys 8 (or 16, 32) further on are a constant away, since
// the turn of the pieces repeats every eight, and block j's address differs in bits 6 and up by j (a
// value's pieces of a block are the low two bits of a piece's number, and stages begin at 512 bytes).
struct Lane {
  int key, value;
};
template <int D>
__device__ __forceinline__ Lane lane_places() {
  using S = Shape<D>;
  static_assert(S::kValuesAt % 512 == 0 && S::kStage % 512 == 0, "block numbers are address bits of their own");
  const int thread = fresh_thread(), lane = thread & 63, half = lane >> 5, l = lane & 15;
  const int dims = S::kHalves == 1 ? 0 : 256 * ((thread >> 6) & 1);  // bytes before the wave's dimensions
  const int value = 16 * piece_at<D>(4 * half + (l >> 2), 2 * ((lane >> 4) & 1) + ((l & 3) >> 1)) + 8 * (l & 1);
  return Lane{(lane & 31) * S::kKeyBytes + 16 * half + dims, S::kValuesAt + (value ^ dims)};
}

typedef __attribute__((address_space(3))) char lds_char;
__device__ __forceinline__ u32x2 read_values(uint32_t at) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_char*)(uintptr_t)at));
}

// A wave's softmax state for its 32 query rows (one per lane column): running maximum, the lane's
// part of the sum, and the unnormalised output of the lane's dimensions.
template <int D>
struct State {
  f32x16 acc[Shape<D>::kBlocks];
  float m, l;
};

// A masked key of a tile may hold infinities or NaN, which a probability of 0 does not cancel in the
// product, while another column sees that key.  The product then takes such values as 0, and they
// are added to the columns that see them (where the sum is no longer finite whatever the weight).
// `seen` is how many of the 32 keys from t0 on the lane column's query row sees.
template <int DT, int D>
__device__ __forceinline__ void add_not_finite(const u32x4* values, State<D>& st, int t0, int seen) {
  constexpr uint32_t kExponent = DT == DS_BF16 ? 0x7f80u : 0x7c00u;
  const int thread = fresh_thread(), half = (thread >> 5) & 1;
  const int first = Shape<D>::kHalves == 1 ? 0 : 16 * ((thread >> 6) & 1);
#pragma unroll 1
  for (int t = 0; t < 32; ++t) {
#pragma unroll
    for (int j = 0; j < Shape<D>::kBlocks; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32x2 v = reinterpret_cast<const u32x2*>(values + piece_at<D>(t0 + t, first + 4 * j + i))[half];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint16_t x = static_cast<uint16_t>(v[e >> 1] >> (16 * (e & 1)));
          if (t < seen && (x & kExponent) == kExponent) st.acc[j][4 * i + e] += Elem<DT>::load(x);
        }
      }
    }
  }
}

// 32 keys of a staged tile for one wave, from key t0 of the tile on.  `seen` (MASKED): how many of
// them the lane column's query row sees, and `poison` that a value of the tile is not finite.  Reads
// of a step are issued together, ahead of the products that take them: the keys' before the first
// product, the values' before the softmax.  All waves of halves (kHalves) come here together, or to
// the same barrier.
template <int DT, int D, bool MASKED>
__device__ __forceinline__ void attend_keys(const char* stage, const Lane& at, const u32x4 (&q)[Shape<D>::kSteps],
                                            State<D>& st, int t0, int seen, bool poison, float scale_log2,
                                            char* scores) {
  using S = Shape<D>;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const char* keys = stage + at.key + t0 * S::kKeyBytes;
  f32x16 sc;
#pragma unroll
  for (int i = 0; i < 16; ++i) sc[i] = 0.f;
  u32x4 k[S::kSteps];
#pragma unroll
  for (int s = 0; s < S::kSteps; ++s) k[s] = *reinterpret_cast<const u32x4*>(keys + 32 * s);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int s = 0; s < S::kSteps; ++s) sc = mfma32<DT>(k[s], q[s], sc);
  if constexpr (S::kHalves == 2) {  // the other half's part of the scores
    const int thread = fresh_thread();
    f32x4* mine = reinterpret_cast<f32x4*>(scores) + (thread >> 6) * 256 + (thread & 63);
    const f32x4* other = reinterpret_cast<const f32x4*>(scores) + ((thread >> 6) ^ 1) * 256 + (thread & 63);
#pragma unroll
    for (int i = 0; i < 4; ++i) mine[64 * i] = f32x4{sc[4 * i], sc[4 * i + 1], sc[4 * i + 2], sc[4 * i + 3]};
    lds_barrier();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 x = other[64 * i];
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[4 * i + e] += x[e];
    }
  }
  u32x2 v[2][S::kBlocks][2];
  const uint32_t values = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const lds_char*)stage)) + at.value;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
#pragma unroll
    for (int j = 0; j < S::kBlocks; ++j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) v[s][j][e] = read_values((values ^ (64 * j)) + (t0 + 16 * s + 8 * e) * 2 * D);
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  float top = -INFINITY;
  // Masked scores are no part of the maximum, and their weights are 0 as such: -infinity times a scale of 0
  // is none.
  auto sees = [&](int i) { return !MASKED || 8 * (i >> 2) + (i & 3) < seen - 4 * half; };
#pragma unroll
  for (int i = 0; i < 16; ++i) top = fmaxf(top, sees(i) ? sc[i] : -INFINITY);
  // The reference of the exponents follows the maximum only when it is 2^8 behind: weights of up to 2^8
  // keep their relative precision, and most tiles leave the sums as they are.  In fp16 it stays 2^7 below
  // the maximum, so that weights lie in 2^-24 .. 2^15 of the type: those of a long tail of small
  // probabilities are then rounded relative to themselves down to 2^-21 of the largest.
  constexpr float kBelow = DT == DS_FP16 ? 7.f : 0.f;
  top = fmaxf(top, other_half(top));
  if (!MASKED || top != -INFINITY) top = __builtin_fmaf(top, scale_log2, -kBelow);
  if (__any(top > st.m + 8.f)) {
    const float m = fmaxf(st.m, top);
    const float keep = st.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.m - m);
    st.m = m;
    st.l *= keep;
#pragma unroll
    for (int j = 0; j < S::kBlocks; ++j) {
#pragma unroll
      for (int i = 0; i < 16; ++i) st.acc[j][i] *= keep;
    }
  }
  const float m = st.m == -INFINITY ? 0.f : st.m;
  u32x4 p[2];
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    const float x = sees(i) ? __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], scale_log2, -m)) : 0.f;
    const float y = sees(i + 1) ? __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i + 1], scale_log2, -m)) : 0.f;
    // The product's operands are 16 bits, so the probabilities are rounded for it; the sum is of them as
    // computed, since the LSE is an fp32 output.
    st.l += x + y;
    p[i >> 3][(i & 7) >> 1] = pack2<DT>(x, y);
  }
  constexpr uint32_t kExponent = DT == DS_BF16 ? 0x7f80u : 0x7c00u;
  // The lane's own probabilities are the B operand: k-slot (half, e) of step s is key 16 s + 8 (e /
  // 4) + 4 half + e % 4 of the 32, and the values are read in that order.
  auto output = [&](int j, int s, u32x2 lo, u32x2 hi) {
    u32x4 x = u32x4{lo[0], lo[1], hi[0], hi[1]};
    if constexpr (MASKED) {
      if (poison) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] &= ((x[e] & kExponent) == kExponent ? 0u : 0xffffu) |
                  ((x[e] & (kExponent << 16)) == (kExponent << 16) ? 0u : 0xffff0000u);
        }
      }
    }
    st.acc[j] = mfma32<DT>(x, p[s], st.acc[j]);
  };
#pragma unroll
  for (int s = 0; s < 2; ++s) {
#pragma unroll
    for (int j = 0; j < S::kBlocks; ++j) output(j, s, v[s][j][0], v[s][j][1]);
  }
  if constexpr (MASKED) {
    if (poison) add_not_finite<DT, D>(reinterpret_cast<const u32x4*>(stage + S::kValuesAt), st, t0, seen);
  }
}

// Pieces in the workspace: for each slot 128 maxima and 128 sums, then the outputs as the waves
// hold them ([query block][4 x dimension group][lane] of 4 floats).
template <int D>
__device__ __forceinline__ float* piece_sums(const PrefixArgs& a, int slot) {
  return a.pieces + static_cast<int64_t>(slot) * (kWideRows * (D + 2));
}

// How a unit's tile lies over the waves: kQ blocks of 32 query rows, kT waves to a block, which share the
// keys of a tile, kN blocks of 32 each.
template <int D, bool WIDE>
struct Split {
  static constexpr int kQ = WIDE ? 4 : 2;
  static constexpr int kT = Shape<D>::kWaves / kQ / Shape<D>::kHalves;
  static_assert(kT > 0 && Shape<D>::kTile % (32 * kT) == 0);
  static constexpr int kN = Shape<D>::kTile / 32 / kT;
};

// A wave's query rows of a unit.
template <int D>
struct Queries {
  u32x4 q[Shape<D>::kSteps];
  int limit;  // keys that the lane column's row sees
  bool any;
};

// Rows past the unit's end take the tensor's first row, and their results are left out.  Nothing here
// waits for the queries unless there is a sign to turn: they arrive while the first tile goes to shared
// memory, behind the keys in flight.
template <int D>
__device__ __forceinline__ void load_queries(const PrefixArgs& a, const RowTables& t, const Unit& u, int block,
                                             Queries<D>& q) {
  using S = Shape<D>;
  const int thread = fresh_thread(), lane = thread & 63, r0 = u.tile * u.tile_rows + 32 * block;
  const QueryRow row = query_row(a, t, u, r0 + (lane & 31));
  q.any = uniform(r0 < u.rows);
  q.limit = row.limit;
  if (!q.any) return;
  const uint16_t* src = a.q + row.token * a.q_row + row.head * a.q_head + 8 * (lane >> 5) +
                        (S::kHalves == 1 ? 0 : 2 * (thread & 64));
#pragma unroll
  for (int s = 0; s < S::kSteps; ++s) q.q[s] = *reinterpret_cast<const u32x4*>(src + 16 * s);
  if (a.q_sign) {
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s) q.q[s] ^= a.q_sign;
  }
}

// The end of a unit (or of the share inside it): its piece.
template <int D, bool WIDE>
__device__ __forceinline__ void finish_unit(const PrefixArgs& a, const Unit& u, int slot, State<D>& st, int wave,
                                            char* lds) {
  using S = Shape<D>;
  constexpr int kT = Split<D, WIDE>::kT;
  const int lane = fresh_thread() & 63, qb = wave / S::kHalves / kT, tb = wave % kT;
  const int dims = S::kHalves == 1 ? 0 : wave & 1;  // which half of them
  const int r0 = u.tile * u.tile_rows + 32 * qb;
  st.l += other_half(st.l);
  // The waves that share query rows join in shared memory, each for its part of the dimensions (in
  // groups of four accumulators, as they are stored).  Every wave lays down all its groups, its own among
  // them: which are its own is then a matter of addresses, not of selecting registers.
  constexpr int kGroups = 4 * S::kBlocks, kMine = kGroups / kT;
  auto group = [&](int g) {
    return f32x4{st.acc[g >> 2][4 * (g & 3)], st.acc[g >> 2][4 * (g & 3) + 1], st.acc[g >> 2][4 * (g & 3) + 2],
                 st.acc[g >> 2][4 * (g & 3) + 3]};
  };
  f32x4 sum[kMine];
  if constexpr (kT == 1) {
#pragma unroll
    for (int g = 0; g < kGroups; ++g) sum[g] = group(g);
  } else {
    // [wave][group][lane], then each wave's m and l.
    static_assert(S::kWaves * (4 * kGroups + 2) * 64 * 4 <= 2 * S::kStage, "the waves' results fit the tiles");
    f32x4* area = reinterpret_cast<f32x4*>(lds);
    float* sums = reinterpret_cast<float*>(area + S::kWaves * kGroups * 64);
    lds_barrier();
    if (r0 < u.rows) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g) area[(wave * kGroups + g) * 64 + lane] = group(g);
      sums[2 * wave * 64 + lane] = st.m;
      sums[(2 * wave + 1) * 64 + lane] = st.l;
    }
    lds_barrier();
    if (r0 < u.rows) {
      float m = -INFINITY, l = 0.f, weight[kT];
#pragma unroll
      for (int w = 0; w < kT; ++w) {
        weight[w] = sums[2 * (qb * kT + w) * 64 + lane];
        m = fmaxf(m, weight[w]);
      }
#pragma unroll
      for (int w = 0; w < kT; ++w) {
        weight[w] = weight[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(weight[w] - m);
        l += sums[(2 * (qb * kT + w) + 1) * 64 + lane] * weight[w];
      }
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        sum[k] = area[(qb * kT * kGroups + tb * kMine + k) * 64 + lane] * weight[0];
#pragma unroll
        for (int w = 1; w < kT; ++w) sum[k] += area[((qb * kT + w) * kGroups + tb * kMine + k) * 64 + lane] * weight[w];
      }
      st.m = m;
      st.l = l;
    }
  }
  if (r0 < u.rows && slot < a.slots) {
    float* sums = piece_sums<D>(a, slot);
    if (lane < 32 && tb == 0 && dims == 0) {
      sums[32 * qb + lane] = st.m;
      sums[kWideRows + 32 * qb + lane] = st.l;
    }
    f32x4* o = reinterpret_cast<f32x4*>(sums + 2 * kWideRows) +
               ((qb * S::kHalves + dims) * kGroups + tb * kMine) * 64 + lane;
#pragma unroll
    for (int k = 0; k < kMine; ++k) o[k * 64] = sum[k];
  }
}

// What a workgroup carries from tile to tile, across units.
template <int D>
struct Pipe {
  Feed<D> feed;
  Step now, ahead;  // the tile in registers, and the one after it, whose pages are looked up
  Staged<D> s;
  int cur;          // the half of shared memory the next tile goes to
};

// The next tile's keys to shared memory; a register is loaded again as soon as its keys are there.
// CHECK: the tile has a mask; `poison` (a word per wave and stage) then says whether one of its values is
// not finite.
template <int DT, int D, bool WHOLE, bool CHECK>
__device__ __forceinline__ const char* next_tile(const PrefixArgs& a, const Plan& p, const RowTables& t, Pipe<D>& pipe,
                                                 int wave, char* lds, int* poison) {
  using S = Shape<D>;
  const int thread = fresh_thread();
  char* stage = lds + pipe.cur * S::kStage;
  const bool tail = pipe.now.key + S::kTile > pipe.now.key_end || __any(pipe.s.bad != 0);
  Staged<D>& s = pipe.s;
  const int bad = s.bad;
  Places at{};
  if constexpr (WHOLE) at = load_places<D>(a, pipe.ahead, s);
  const int bad_ahead = s.bad;
  bool found = false;
#pragma unroll
  for (int i = 0; i < S::kPasses; ++i) {
    if constexpr (WHOLE) s.bad = bad;
    found |= store_keys<DT, D, CHECK>(a, stage, pipe.now, tail, thread, wave, i, s);
    load_keys<D, WHOLE>(a, pipe.ahead, at, thread, wave, i, s);
  }
  if constexpr (WHOLE) s.bad = bad_ahead;
  if constexpr (CHECK) {
    const int any = __any(found);
    if ((thread & 63) == 0) poison[pipe.cur * S::kWaves + wave] = any;
  }
  pipe.now = pipe.ahead;
  pipe.ahead = pipe.feed.next(a, p, t);
  find_pages<D, WHOLE>(a, pipe.ahead, wave, s);
  pipe.cur ^= 1;
  lds_barrier();
  return stage;
}

// The share's tiles of a unit, from `place` on to `stop`.  Wide and narrow units share the loops: the keys
// in flight stay in their registers from one unit to the next, whatever its kind.
template <int DT, int D, bool WHOLE>
__device__ __forceinline__ void run_unit(const PrefixArgs& a, const Plan& p, const RowTables& t, const Unit& u,
                                         int place, int stop, int group, int wave, Pipe<D>& pipe, char* lds,
                                         char* scores, int* poison) {
  using S = Shape<D>;
  using Wide = Split<D, true>;
  using Narrow = Split<D, S::kHalves == 2>;
  const bool wide = S::kHalves == 2 || u.tile_rows == kWideRows;
  const int first = wide ? 32 * (wave % Wide::kT) * Wide::kN : 32 * (wave % Narrow::kT) * Narrow::kN;
  Queries<D> q;
  load_queries<D>(a, t, u, wave / S::kHalves / (wide ? Wide::kT : Narrow::kT), q);
  State<D> st;
#pragma unroll
  for (int j = 0; j < S::kBlocks; ++j) {
#pragma unroll
    for (int i = 0; i < 16; ++i) st.acc[j][i] = 0.f;
  }
  st.m = -INFINITY;
  st.l = 0.f;
  // Tiles that all query rows see whole, then the ones with a mask.
  for (; place < stop && pipe.now.key + S::kTile <= u.seen_by_all; ++place) {
    const char* stage = next_tile<DT, D, WHOLE, false>(a, p, t, pipe, wave, lds, poison);
    if (q.any) {
      const Lane at = lane_places<D>();
#pragma unroll
      for (int n = 0; n < Wide::kN; ++n) {
        if (n >= Narrow::kN && !wide) break;
        attend_keys<DT, D, false>(stage, at, q.q, st, first + 32 * n, 32, false, a.scale_log2, scores);
      }
    } else if constexpr (S::kHalves == 2) {
      lds_barrier();  // the one in attend_keys
    }
  }
  for (; place < stop; ++place) {
    const int seen = min(q.limit, u.key_end) - pipe.now.key, keys = u.key_end - pipe.now.key;
    const char* stage = next_tile<DT, D, WHOLE, true>(a, p, t, pipe, wave, lds, poison);
    if (q.any) {
      const Lane at = lane_places<D>();
      const bool bad = __any(poison[(pipe.cur ^ 1) * S::kWaves + fresh_thread() % S::kWaves] != 0);
      const int end = min(first + 32 * (wide ? Wide::kN : Narrow::kN), keys);
#pragma unroll 1
      for (int t0 = first; t0 < end; t0 += 32) {
        attend_keys<DT, D, true>(stage, at, q.q, st, t0, seen - t0, bad, a.scale_log2, scores);
      }
    } else if constexpr (S::kHalves == 2) {
      if (keys > 0) lds_barrier();
    }
  }
  lds_barrier();
  if (wide) finish_unit<D, true>(a, u, u.index + group, st, wave, lds);
  else finish_unit<D, S::kHalves == 2>(a, u, u.index + group, st, wave, lds);
  lds_barrier();
}

template <int DT, int D, bool WHOLE>
__global__ __launch_bounds__(Shape<D>::kThreads, 2) void prefix_attention_kernel(PrefixArgs a) {
  using S = Shape<D>;
  __shared__ __attribute__((aligned(512))) char lds[2 * S::kStage];
  __shared__ __attribute__((aligned(16))) char scores[S::kScores ? S::kScores : 16];
  __shared__ RowTables tables;
  __shared__ Plan p;  // read again at each unit
  __shared__ int poison[2 * S::kWaves];
  {
    const Plan made = make_plan<D, S::kThreads>(a, tables, blockIdx.x == 0);
    if (threadIdx.x == 0) p = made;
    __syncthreads();
  }
  // Consecutive shares on one XCD (workgroups are dealt to the eight in turn).
  const int per_xcd = a.groups / 8;
  const int group = a.groups % 8 == 0 ? static_cast<int>(blockIdx.x % 8) * per_xcd + static_cast<int>(blockIdx.x / 8)
                                      : static_cast<int>(blockIdx.x);
  const int wave = uniform(threadIdx.x >> 6), share = uniform(p.share), work = uniform(p.work);
  // Four tiles are under way at a time: one is attended to, the keys of the next are in shared memory or
  // on their way to it, those of the third on their way to registers, the pages of the fourth are looked
  // up.  The order goes across units, so that the memory does not wait for a unit's end.
  Pipe<D> pipe;
  pipe.feed.at = min(group * share, work);
  pipe.feed.end = min(pipe.feed.at + share, work);
  if (pipe.feed.at >= pipe.feed.end) return;
  pipe.feed.start(a, p, tables);
  int place = pipe.feed.at;
  const int end = pipe.feed.end;
  if (place >= end) return;  // the share ends before its unit's first key tile
  Unit u = pipe.feed.unit;
  pipe.cur = 0;
  pipe.s.page = pipe.s.in = pipe.s.bad = 0;
  pipe.now = pipe.feed.next(a, p, tables);
  find_pages<D, WHOLE>(a, pipe.now, wave, pipe.s);
  {
    Places at{};
    if constexpr (WHOLE) at = load_places<D>(a, pipe.now, pipe.s);
#pragma unroll
    for (int i = 0; i < S::kPasses; ++i) load_keys<D, WHOLE>(a, pipe.now, at, threadIdx.x, wave, i, pipe.s);
  }
  pipe.ahead = pipe.feed.next(a, p, tables);
  find_pages<D, WHOLE>(a, pipe.ahead, wave, pipe.s);
  for (;;) {
    place = max(place, u.first_tile);
    const int stop = min(end, u.first_tile + u.key_tiles);
    if (place >= stop) return;  // the share ends before the unit's first key tile
    run_unit<DT, D, WHOLE>(a, p, tables, u, place, stop, group, wave, pipe, lds, scores, poison);
    place = stop;
    if (place >= end) return;
    u = unit_at<D>(a, p, tables, place);
  }
}

// Joins the pieces of 32 query rows of one KV head (the batch's order) for 32 dimensions: eight waves
// take the pieces in turn, and the first four join the waves' sums, four dimensions of a lane each.
// Latency-bound.  Both kernels in us for two rows over 1 k keys, 16 over 16 k, 80 query tokens over 32 k and 57
// ragged rows over 5 k: 15.2, 38.8, 86.5, 71.3; with four waves 16.0, 41.1, 86.1, 70.1, with 16 16.0, 38.7, 90.8, 79.4.
constexpr int kJoinWaves = 8;
template <int DT, int D>
__global__ __launch_bounds__(64 * kJoinWaves) void prefix_join_kernel(PrefixArgs a) {
  __shared__ RowTables tables;
  __shared__ float joined[kJoinWaves][18][64];
  const Plan p = make_plan<D, 64 * kJoinWaves>(a, tables, false);
  const int rows = p.query_tokens * a.group;
  const int block = blockIdx.x, j = blockIdx.y, h = blockIdx.z;
  if (32 * block >= rows) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r = 32 * block + (lane & 31);
  const bool valid = r < rows;
  const int token = (valid ? r : rows - 1) / a.group;
  const int b = row_at(a, tables, token), i = token - tables.token[b];

  float m = -INFINITY, l = 0.f;
  f32x4 acc[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) acc[k] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto join = [&](int slot, int row_in_tile) {
    const float* sums = piece_sums<D>(a, slot);
    const float om = sums[row_in_tile], ol = sums[kWideRows + row_in_tile];
    const f32x4* o = reinterpret_cast<const f32x4*>(sums + 2 * kWideRows) +
                     ((row_in_tile >> 5) * (D / 32) + j) * 4 * 64 + (row_in_tile & 31) + (lane & 32);
    f32x4 part[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) part[k] = o[k * 64];
    const float top = fmaxf(m, om);
    const float mine = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    const float other = om == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(om - top);
    m = top;
    l = l * mine + ol * other;
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] = acc[k] * mine + part[k] * other;
  };
  // A segment is about a share long: its pieces are of one workgroup or of two, seldom of more.
  const int tile = 32 * block / p.prefix_tile, in_tile = 32 * block - tile * p.prefix_tile + (lane & 31);
  for (int k = wave; k < 2 * p.segments; k += kJoinWaves) {
    const Unit u = prefix_unit<D>(a, p, h, k >> 1, tile);
    const int last = (u.first_tile + u.key_tiles - 1) / p.share;
    for (int group = u.first_tile / p.share + (k & 1); group <= last; group += 2) join(u.index + group, in_tile);
  }
  if (tables.work[b + 1] > tables.work[b]) {
    const int in_row = i * a.group + (valid ? r : rows - 1) % a.group;
    const int n = tile_rows<D>((tables.token[b + 1] - tables.token[b]) * a.group);
    const Unit u = own_unit<D>(a, p, tables, b, h, in_row / n);
    const int last = (u.first_tile + u.key_tiles - 1) / p.share;
    for (int group = u.first_tile / p.share + wave; group <= last; group += kJoinWaves) {
      join(u.index + group, in_row % n);
    }
  }
  joined[wave][16][lane] = m;
  joined[wave][17][lane] = l;
#pragma unroll
  for (int k = 0; k < 16; ++k) joined[wave][k][lane] = acc[k >> 2][k & 3];
  __syncthreads();
  if (wave >= 4 || !valid) return;
  m = joined[0][16][lane];
  for (int w = 1; w < kJoinWaves; ++w) m = fmaxf(m, joined[w][16][lane]);
  l = 0.f;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  for (int w = 0; w < kJoinWaves; ++w) {
    const float om = joined[w][16][lane];
    const float weight = om == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(om - m);
    l += joined[w][17][lane] * weight;
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] += joined[w][4 * wave + k][lane] * weight;
  }
  const int head = h * a.group + r % a.group;
  const int64_t q_token = static_cast<int64_t>(tables.start[b]) + i;
  x *= l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;  // nothing seen: zeros; NaN stays NaN
  uint16_t* out = a.out + q_token * a.o_row + head * a.o_head + 32 * j + 8 * wave + 4 * (lane >> 5);
  *reinterpret_cast<u32x2*>(out) = u32x2{pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3])};
  if (a.lse && j == 0 && wave == 0 && lane < 32) {
    a.lse[q_token * a.l_row + head * a.l_head] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2P;
  }
}

int attention_groups() { return device_cu_count(); }

// Pieces of a launch: units of the prefix (at most a segment per workgroup and one per tile of query
// rows), units of the rows, and one more per workgroup where a share ends inside a unit.
int64_t piece_slots(int rows, int tokens, int num_q_heads, int num_kv_heads) {
  const int64_t query_rows = static_cast<int64_t>(tokens) * (num_q_heads / num_kv_heads);
  const int64_t tiles = query_rows / kNarrowRows + 1;
  return 2 * static_cast<int64_t>(attention_groups()) + num_kv_heads * (2 * tiles + rows);
}

template <int DT, int D>
int launch(hipStream_t stream, const PrefixArgs& a) {
  const bool whole = a.block_size % Shape<D>::kPerLoad == 0;
  if (whole) prefix_attention_kernel<DT, D, true><<<a.groups, Shape<D>::kThreads, 0, stream>>>(a);
  else prefix_attention_kernel<DT, D, false><<<a.groups, Shape<D>::kThreads, 0, stream>>>(a);
  const int blocks = static_cast<int>((static_cast<int64_t>(a.tokens) * a.group + 31) / 32);
  prefix_join_kernel<DT, D><<<dim3(blocks, D / 32, a.hkv), 64 * kJoinWaves, 0, stream>>>(a);
  return check_launch("ds_prefix_attention");
}

template <int DT>
int launch_dim(hipStream_t stream, int d, const PrefixArgs& a) {
  if (d == 64) return launch<DT, 64>(stream, a);
  if (d == 128) return launch<DT, 128>(stream, a);
  return launch<DT, 256>(stream, a);
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

size_t workspace_bytes(int rows, int tokens, int num_q_heads, int num_kv_heads, int head_dim) {
  if (rows <= 0 || tokens <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads) return 0;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 0;
  return static_cast<size_t>(piece_slots(rows, tokens, num_q_heads, num_kv_heads)) * kWideRows *
         (head_dim + 2) * sizeof(float);
}

int prefix_attention_impl(hipStream_t stream, const ds_prefix_attention_desc* d) {
  DS_REQUIRE(d != nullptr, "null descriptor");
  DS_REQUIRE(d->dtype == DS_BF16 || d->dtype == DS_FP16, "queries and KV caches must use BF16 or FP16");
  DS_REQUIRE(d->rows >= 0 && d->tokens >= 0, "row and token counts must be non-negative");
  DS_REQUIRE(d->num_q_heads > 0 && d->num_kv_heads > 0 && d->num_q_heads % d->num_kv_heads == 0,
             "query heads must be divisible by KV heads");
  DS_SUPPORTED(d->head_dim == 64 || d->head_dim == 128 || d->head_dim == 256, "head_dim must be 64, 128 or 256");
  DS_SUPPORTED(d->rows <= kMaxRows, "at most %d rows", kMaxRows);
  DS_REQUIRE(d->block_size > 0 && d->num_blocks > 0 && d->max_blocks > 0, "block sizes and counts must be positive");
  DS_SUPPORTED(d->block_size <= (1 << 20), "at most 2^20 tokens per page");
  if (d->rows == 0 || d->tokens == 0) return clear_error();
  DS_REQUIRE(d->query && d->output && d->key_cache && d->value_cache && d->block_table && d->query_start &&
                 d->query_len && d->target_len && d->prefix_len,
             "null tensor pointer");
  const int64_t strides[] = {d->q_row_stride,   d->q_head_stride,  d->o_row_stride,   d->o_head_stride, d->k_block_stride,
                             d->k_token_stride, d->k_head_stride,  d->v_block_stride, d->v_token_stride, d->v_head_stride};
  for (int64_t s : strides) DS_REQUIRE(s >= 0 && s % 8 == 0, "row, page and head strides must be multiples of 8 elements");
  // Places within a page are 32-bit byte counts.
  const int64_t in_key = d->k_block_stride + d->block_size * d->k_token_stride + d->num_kv_heads * d->k_head_stride;
  const int64_t in_value = d->v_block_stride + d->block_size * d->v_token_stride + d->num_kv_heads * d->v_head_stride;
  DS_SUPPORTED(d->k_block_stride < (1 << 30) && d->v_block_stride < (1 << 30) && d->k_token_stride < (1 << 30) &&
                   d->v_token_stride < (1 << 30) && d->k_head_stride < (1 << 30) && d->v_head_stride < (1 << 30) &&
                   in_key < (1 << 30) && in_value < (1 << 30),
               "pages of at most 2^30 elements");
  DS_REQUIRE(aligned(d->query) && aligned(d->output) && aligned(d->key_cache) && aligned(d->value_cache),
             "query, output and KV caches must be 16-byte aligned");
  const size_t need = workspace_bytes(d->rows, d->tokens, d->num_q_heads, d->num_kv_heads, d->head_dim);
  DS_REQUIRE(d->workspace && d->workspace_bytes >= need && (reinterpret_cast<uintptr_t>(d->workspace) & 255u) == 0,
             "workspace must be 256-byte aligned and hold ds_prefix_attention_workspace_bytes()");
  const int group = d->num_q_heads / d->num_kv_heads;
  const int64_t capacity = std::min<int64_t>(static_cast<int64_t>(d->max_blocks) * d->block_size, 1 << 30);
  const int tile = tile_keys(d->head_dim);
  const int64_t tiles = static_cast<int64_t>(d->tokens) * group / kNarrowRows + 1 + d->rows;
  DS_SUPPORTED(d->tokens <= (1 << 20), "at most 2^20 query tokens");
  // The places of the work (own and prefix tiles, and their costs) are counted in 32 bits.
  const int64_t places = (capacity + tile - 1) / tile + 2 * unit_cost(d->head_dim) + 2;
  DS_SUPPORTED(d->num_kv_heads * tiles * places * 2 < INT_MAX &&
                   static_cast<int64_t>(d->tokens) * group < INT_MAX / 2 && d->num_kv_heads <= 65535,
               "too many query tokens, KV heads or keys for one launch");
  PrefixArgs a{};
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
  a.capacity = static_cast<int>(capacity);
  a.num_blocks = d->num_blocks;
  a.block_size = d->block_size;
  a.per_block = 1.f / static_cast<float>(d->block_size);
  a.q_start = d->query_start, a.q_len = d->query_len, a.t_len = d->target_len, a.prefix_len = d->prefix_len;
  a.rows = d->rows, a.tokens = d->tokens, a.hkv = d->num_kv_heads, a.group = group;
  a.scale_log2 = std::fabs(d->scale) * kLog2eP;
  a.q_sign = d->scale < 0.f ? 0x80008000u : 0u;
  a.pieces = static_cast<float*>(d->workspace);
  a.slots = static_cast<int>(piece_slots(d->rows, d->tokens, d->num_q_heads, d->num_kv_heads));
  a.groups = attention_groups();
  a.status = d->status;
  return d->dtype == DS_BF16 ? launch_dim<DS_BF16>(stream, d->head_dim, a) : launch_dim<DS_FP16>(stream, d->head_dim, a);
}

}  // namespace
}  // namespace ds355

extern "C" size_t ds_prefix_attention_workspace_bytes(int rows, int tokens, int num_q_heads, int num_kv_heads,
                                                      int head_dim) {
  return ds355::workspace_bytes(rows, tokens, num_q_heads, num_kv_heads, head_dim);
}

extern "C" int ds_prefix_attention(ds_stream_t stream, const ds_prefix_attention_desc* desc) {
  return ds355::prefix_attention_impl(reinterpret_cast<hipStream_t>(stream), desc);
}

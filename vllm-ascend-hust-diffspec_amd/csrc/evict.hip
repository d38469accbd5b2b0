// Eviction from a paged cache: each KV head of a row keeps its keep_len[b] best slots, in place.
//
// A row's slots are its tokens' places in its pages; positions[b, h, t] says which token of the request a
// slot holds once an eviction has moved tokens, and slots at or past settled[b][0] still hold theirs in
// order: token t + settled[b][1], where settled[b][1] tokens have been evicted before.  Of n =
// target_len[b] slots a head keeps k = keep_len[b]:
//
//   - those of the first `sinks` tokens and of the newest `recent` ones,
//   - then those of largest mass, ties to the lowest slot (NaN counts as less than any number).
//
// The kept slots below k stay.  The j-th kept slot at or past k moves to the j-th slot below k that is not
// kept: sources and destinations are apart, so the moves run in any order, in place, and a step that evicts
// one token moves one token.
//
// evict_select_kernel: a workgroup a (row, KV head), which holds up to 32 k values in shared memory, as integers
// of the same order.  The k-th largest is found 11 bits at a time from histograms in shared memory, after the
// first 11 among the few that share them.  Slots that are always kept and masses of 0, of which there may be many
// alike, are counted by the lanes instead of by atomics on one word.  It leaves, for every 64 slots, which
// are kept and how many slots to move to and from lie before them.
//
// evict_move_kernel: a workgroup takes 64 of a head's moves at a time, finds their slots from those counts, and
// moves keys, values, masses and positions.  Slots that do not move get their masses and positions here as well,
// where there are many workgroups.
//
// What bounds it: the selection is one CU's work for a head, in a handful of dependent passes before any move (10 us
// for 2049 slots, 27 for 28 k, of which the search takes 9); long heads' moves run at the rate of a large copy.  4 rows of
// 20 k to 32 k slots, 8 heads of 128 dimensions, cut to 4096: 67 us; one token too many in 16 rows of 2049: 16.5 us.
#include "matrix.h"

namespace ds355 {
namespace {

constexpr uint32_t kStatusLength = 2;   // a row is longer than its block table, mass or positions
constexpr uint32_t kStatusPage = 4;     // a page id is out of range
constexpr uint32_t kStatusBudget = 8;   // keep_len is negative, or less than the tokens that are always kept
constexpr uint32_t kStatusShared = 16;  // a page that would be written is shared

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / 64;
constexpr int kMoveThreads = 256;

// What a head leaves for its moves (-1: the row is left alone), and the row's state before them.
struct Head {
  int moves, known, gone, groups;
};
// 64 slots of a head: which are kept, and how many holes and movers lie before them.
struct Group {
  uint64_t kept;
  int holes, movers;
};

struct EvictArgs {
  char* k;
  int64_t k_block, k_token, k_head;  // bytes
  char* v;
  int64_t v_block, v_token, v_head;
  float* mass;
  int64_t m_row, m_head;
  int32_t* positions;
  int64_t p_row, p_head;
  int32_t* settled;  // [rows][2]
  const int32_t* table;
  int64_t bt_stride;
  const int32_t* ref_counts;  // or null
  const int32_t* t_len;
  const int32_t* keep_len;
  int32_t* kept_len;
  int capacity;
  int num_blocks, block_size;
  int rows, hkv, pieces;  // pieces: 16-byte pieces of a head's key
  int sinks, recent;
  int groups;         // of 64 slots, of a head at most
  Head* heads;    // [rows * hkv]
  Group* lists;   // [rows * hkv][groups]
  int32_t* status;
};

// Unsigned integers in the order of floating-point values; NaN below all, and 0 for no slot.
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 1;
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ void report(const EvictArgs& a, uint32_t bits) {
  if (a.status) __hip_atomic_fetch_or(a.status, static_cast<int>(bits), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

constexpr uint32_t kAlways = 0xffffffffu;  // above every mass
constexpr uint32_t kZero = 0x80000000u;    // a mass of 0
constexpr int kBins = 2048;

constexpr int kFew = 4096;  // values that share their first bits, held in shared memory

// Sum over the waves before, and over all (`all`), of a count that is the same in a wave's lanes.
__device__ __forceinline__ int wave_prefix(int count, int* scratch, int& all) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  __syncthreads();
  if (lane == 0) scratch[wave] = count;
  __syncthreads();
  const int mine = lane < kSelectWaves ? scratch[lane] : 0, inclusive = wave_inclusive_scan(mine);
  all = __builtin_amdgcn_readlane(inclusive, 63);
  return __builtin_amdgcn_readlane(inclusive - mine, uniform(wave));
}

// The i-th set bit of `bits`, which has more.
__device__ __forceinline__ int set_bit(uint64_t bits, int i) {
  int at = 0;
#pragma unroll
  for (int width = 32; width >= 1; width >>= 1) {
    const int low = __popcll((bits >> at) & ((1ull << width) - 1));
    if (i >= low) i -= low, at += width;
  }
  return at;
}

// HELD: slots whose values are held in shared memory; those of a longer row are read again for every pass.  The least
// that holds the longest row is taken, so that more workgroups fit a CU: 57 rows of up to 6000 slots, 8 heads, take
// 68 us with 8192 and 73 with 32768, 16 rows of 2049, 4 heads, 16.5 with 4096 and 16.8.
template <int HELD>
__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(EvictArgs a) {
  constexpr int kGroups = HELD / 64;  // of 64 slots, a wave's
  static_assert(kGroups <= kSelectThreads && HELD < 65536, "a thread a group; two counts of a chunk in a word");
  __shared__ uint32_t values[HELD];
  __shared__ __attribute__((aligned(16))) int histogram[kBins];
  __shared__ uint32_t few[kFew];
  __shared__ int scratch[kSelectWaves];
  struct Masks {
    uint64_t more, equal;  // of a group's slots: values above the least kept one, and like it
  };
  static_assert(kGroups * sizeof(Masks) <= sizeof(histogram), "where the histogram was");
  Masks* masks = reinterpret_cast<Masks*>(histogram);
  __shared__ int found, left, share, refused, few_held;
  const int b = blockIdx.x / a.hkv, h = blockIdx.x - b * a.hkv;
  const int tid = threadIdx.x, lane = tid & 63;
  const int n = a.t_len[b], keep = a.keep_len[b];
  uint32_t bits = 0;
  if (n > a.capacity) {
    bits = kStatusLength;
  } else if (n > 0 && (keep < 0 || (keep < n && a.sinks > keep - a.recent))) {
    bits = kStatusBudget;
  }
  const bool asked = !bits && n > keep && n > 0;
  float* mass = a.mass + b * a.m_row + h * a.m_head;
  int32_t* positions = a.positions + b * a.p_row + h * a.p_head;
  const int known = min(max(a.settled[2 * b], 0), n), gone = a.settled[2 * b + 1];
  const int newest = n + gone - a.recent;  // tokens at or past it are always kept
  auto position = [&](int t) { return t < known ? positions[t] : t + gone; };
  auto value_of = [&](int place, float weight) { return place < a.sinks || place >= newest ? kAlways : ordered(weight); };
  // f(slot, value) for the slots from `first` on, one a thread and 1024 apart, and none (0) past the last one, in
  // whole waves.
  auto each = [&](int first, int end, auto f) {
    int t = first + tid;
    for (; t - lane < min(end, HELD); t += kSelectThreads) f(t, t < n ? values[t] : 0u);
    for (; t - lane < end; t += kSelectThreads) f(t, t < n ? value_of(position(t), mass[t]) : 0u);
  };
  if (tid == 0) refused = 0, few_held = 0;
  for (int i = tid; i < kBins; i += kSelectThreads) histogram[i] = 0;
  constexpr int kFirst = 21;  // the first histogram is of the bits from it on
  auto counted = [](uint32_t x) { return x - 1 < kAlways - 1 && x != kZero; };
  int always = 0, zeros = 0;
  auto count_first = [&](uint32_t x) {
    always += x == kAlways;
    zeros += x == kZero;
    if (counted(x)) atomicAdd(&histogram[x >> kFirst], 1);
  };
  __syncthreads();
  if (asked) {
    // Eight loads of a thread are under way before the first is looked at.
    const int last = min(n, HELD) - 1;
    for (int first = tid; first <= last; first += 8 * kSelectThreads) {
      float weight[8];
      int place[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) weight[i] = mass[min(first + i * kSelectThreads, last)];
#pragma unroll
      for (int i = 0; i < 8; ++i) place[i] = position(min(first + i * kSelectThreads, last));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (first + i * kSelectThreads <= last) {
          const uint32_t x = value_of(place[i], weight[i]);
          values[first + i * kSelectThreads] = x;
          count_first(x);
        }
      }
    }
    for (int i = tid; i < ceil_div(n, a.block_size); i += kSelectThreads) {
      const int page = a.table[b * a.bt_stride + i];
      if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.num_blocks)) {
        atomicOr(&refused, kStatusPage);
      } else if (a.ref_counts && i * a.block_size < keep && a.ref_counts[page] > 1) {
        atomicOr(&refused, kStatusShared);
      }
    }
  }
  if (asked) each(HELD, n, [&](int, uint32_t x) { count_first(x); });
  wave_prefix(wave_total(always), scratch, always);
  wave_prefix(wave_total(zeros), scratch, zeros);
  bits |= refused;
  const bool work = asked && !bits;
  if (tid == 0) {
    if (h == 0) a.kept_len[b] = work ? keep : max(n, 0);
    if (!work) a.heads[blockIdx.x].moves = -1;
    if (bits && h == 0) report(a, bits);
  }
  if (!work) return;

  // The least kept value and how many of its equals are kept (all of them where a whole class is).
  uint32_t value = kAlways;
  int need = keep == always ? INT_MAX : keep;
  if (always < keep) {
    value = 0;
    need = keep - always;  // kept values among those that share the bits found so far
    bool in_few = false;
    for (int high = 32, shift = kFirst; ; high = shift, shift = max(shift - 11, 0)) {
      auto shares = [&](uint32_t x) { return high == 32 || (x >> high) == (value >> high); };
      auto bin = [&](uint32_t x) { return (x >> shift) & ((1 << (high - shift)) - 1); };
      if (high < 32) {
        for (int i = tid; i < kBins; i += kSelectThreads) histogram[i] = 0;
        __syncthreads();
        auto count = [&](uint32_t x) {
          if (counted(x) && shares(x)) atomicAdd(&histogram[bin(x)], 1);
        };
        if (in_few) {
          for (int i = tid; i < few_held; i += kSelectThreads) count(few[i]);
        } else {
          each(0, n, [&](int, uint32_t x) { count(x); });
        }
      }
      if (tid == 0 && zeros && shares(kZero)) atomicAdd(&histogram[bin(kZero)], zeros);
      __syncthreads();
      // Bins from the largest down, two a thread.
      const int first = histogram[kBins - 1 - 2 * tid], second = histogram[kBins - 2 - 2 * tid];
      const int inclusive = wave_inclusive_scan(first + second);
      int all;
      const int above = wave_prefix(__builtin_amdgcn_readlane(inclusive, 63), scratch, all) + inclusive - first - second;
      if (above < need && need <= above + first) {
        found = kBins - 1 - 2 * tid, left = need - above, share = first;
      } else if (above + first < need && need <= above + first + second) {
        found = kBins - 2 - 2 * tid, left = need - above - first, share = second;
      }
      __syncthreads();
      value |= static_cast<uint32_t>(found) << shift;
      need = left;
      const int sharing = share;
      if (need == sharing) need = INT_MAX;
      if (need == INT_MAX || shift == 0) break;
      if (high == 32 && sharing <= kFew) {  // (masses of 0 among them are counted apart)
        in_few = true;
        each(0, n, [&](int, uint32_t x) {
          if (counted(x) && (x >> kFirst) == (value >> kFirst)) few[atomicAdd(&few_held, 1)] = x;
        });
      }
      __syncthreads();
    }
  }
  value = max(value, 1u);  // no slots have 0
  if (keep == 0) value = kAlways, need = 0;

  // Slots in order, group by group: a scan over the groups' counts says what lies before each.
  Group* list = a.lists + static_cast<int64_t>(blockIdx.x) * a.groups;
  int ties = 0, holes = 0, movers = 0;  // of the chunks before
  constexpr int kChunk = 64 * kGroups;
  for (int first = 0; first < n; first += kChunk) {
    const int end = min(first + kChunk, n);
    __syncthreads();
    each(first, end, [&](int t, uint32_t x) {
      const uint64_t more = __ballot(x > value), equal = __ballot(x == value);
      if (lane == 0) masks[(t - first) >> 6] = Masks{more, equal};
    });
    __syncthreads();
    const bool mine = tid < ceil_div(end - first, 64);  // a thread a group
    const Masks m = mine ? masks[tid] : Masks{0, 0};
    const int equal = __popcll(m.equal), inclusive = wave_inclusive_scan(equal);
    int ties_here;
    const int before = ties + wave_prefix(__builtin_amdgcn_readlane(inclusive, 63), scratch, ties_here) + inclusive - equal;
    const int take = need - before;  // of the values like the least kept one
    const uint64_t kept =
        m.more | (take >= equal ? m.equal : take <= 0 ? 0 : m.equal & ((1ull << set_bit(m.equal, take)) - 1));
    const int low_slots = keep - (first + 64 * tid);  // slots below `keep` exist
    const uint64_t low = low_slots >= 64 ? ~0ull : low_slots <= 0 ? 0ull : (1ull << low_slots) - 1;
    // Holes, and movers in the upper half.
    const int moves = mine ? __popcll(low & ~kept) | __popcll(kept & ~low) << 16 : 0;
    const int moves_inclusive = wave_inclusive_scan(moves);
    int moves_here;
    const uint32_t moves_before =
        wave_prefix(__builtin_amdgcn_readlane(moves_inclusive, 63), scratch, moves_here) + moves_inclusive - moves;
    if (mine) {
      list[first / 64 + tid] =
          Group{kept, holes + static_cast<int>(moves_before & 0xffff), movers + static_cast<int>(moves_before >> 16)};
    }
    ties += ties_here, holes += moves_here & 0xffff, movers += static_cast<uint32_t>(moves_here) >> 16;
  }
  if (tid == 0) a.heads[blockIdx.x] = Head{holes, known, gone, ceil_div(n, 64)};  // as many movers as holes
}

constexpr int kMoves = 64;         // moves of a workgroup at a time
constexpr int kMostSearched = 512;  // groups whose counts are searched in shared memory

__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a) {
  __shared__ int2 moves[kMoves];
  __shared__ int2 before[kMostSearched];  // holes and movers before a group
  const Head head = a.heads[blockIdx.y];
  if (head.moves < 0) return;
  const int b = blockIdx.y / a.hkv, h = blockIdx.y - b * a.hkv, keep = a.keep_len[b], tid = threadIdx.x;
  if (h == 0 && blockIdx.x == 0 && tid == 0) {
    a.settled[2 * b + 1] = head.gone + a.t_len[b] - keep;
    a.settled[2 * b] = keep;
  }
  const Group* list = a.lists + static_cast<int64_t>(blockIdx.y) * a.groups;
  float* mass = a.mass + b * a.m_row + h * a.m_head;
  int32_t* positions = a.positions + b * a.p_row + h * a.p_head;
  // Slots that do not move: those given up lose their mass, and kept ones get their positions.
  constexpr int kWaves = kMoveThreads / 64;
  const int n = a.t_len[b], lane = tid & 63;
  for (int g = min(head.known, keep) / 64 + blockIdx.x * kWaves + (tid >> 6); g < head.groups; g += gridDim.x * kWaves) {
    const int t = 64 * g + lane;
    const bool kept = list[g].kept >> lane & 1;
    if (t >= keep) {
      if (!kept && t < n) mass[t] = 0.f;
    } else if (kept && t >= head.known) {
      positions[t] = t + head.gone;
    }
  }
  if (static_cast<int>(blockIdx.x) * kMoves >= head.moves) return;
  const bool shared = head.groups <= kMostSearched;
  if (shared) {
    for (int g = tid; g < head.groups; g += kMoveThreads) before[g] = int2{list[g].holes, list[g].movers};
  }
  const int32_t* pages = a.table + b * a.bt_stride;
  for (int first = blockIdx.x * kMoves; first < head.moves; first += gridDim.x * kMoves) {
    const int count = min(kMoves, head.moves - first);
    __syncthreads();
    // Threads 0 to 63 find the slots that are moved to, 64 to 127 those that are moved from.
    const int i = tid % kMoves;
    if (tid < 2 * kMoves && i < count) {
      const bool from = tid >= kMoves;
      int lo = 0, hi = head.groups - 1;  // the last group with no more of them before it
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        const int2 x = shared ? before[mid] : int2{list[mid].holes, list[mid].movers};
        if ((from ? x.y : x.x) <= first + i) lo = mid; else hi = mid - 1;
      }
      const Group g = list[lo];
      const int low_slots = keep - 64 * lo;
      const uint64_t low = low_slots >= 64 ? ~0ull : low_slots <= 0 ? 0ull : (1ull << low_slots) - 1;
      const int t = 64 * lo + set_bit(from ? g.kept & ~low : low & ~g.kept, first + i - (from ? g.movers : g.holes));
      if (from) moves[i].x = t; else moves[i].y = t;
    }
    __syncthreads();
    if (tid < count) {
      const int2 m = moves[tid];
      const float weight = mass[m.x];
      positions[m.y] = m.x < head.known ? positions[m.x] : m.x + head.gone;
      mass[m.y] = weight;
      mass[m.x] = 0.f;
    }
    for (int j = tid; j < count * a.pieces; j += kMoveThreads) {
      const int move = j / a.pieces, piece = j - move * a.pieces;
      const int2 m = moves[move];
      const int from = m.x / a.block_size, to = m.y / a.block_size;
      const int64_t source = pages[from], target = pages[to];
      const int in_from = m.x - from * a.block_size, in_to = m.y - to * a.block_size;
      const u32x4 key =
          *reinterpret_cast<const u32x4*>(a.k + source * a.k_block + in_from * a.k_token + h * a.k_head + 16 * piece);
      const u32x4 value =
          *reinterpret_cast<const u32x4*>(a.v + source * a.v_block + in_from * a.v_token + h * a.v_head + 16 * piece);
      *reinterpret_cast<u32x4*>(a.k + target * a.k_block + in_to * a.k_token + h * a.k_head + 16 * piece) = key;
      *reinterpret_cast<u32x4*>(a.v + target * a.v_block + in_to * a.v_token + h * a.v_head + 16 * piece) = value;
    }
  }
}

size_t rounded(size_t n) { return (n + 255) & ~size_t{255}; }

size_t evict_workspace_bytes(int rows, int num_kv_heads, int capacity) {
  if (rows <= 0 || num_kv_heads <= 0 || capacity <= 0) return 0;
  const size_t heads = static_cast<size_t>(rows) * num_kv_heads;
  return rounded(heads * sizeof(Head)) + heads * ((capacity + 63) / 64) * sizeof(Group);
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int evict_impl(hipStream_t stream, const ds_evict_desc* d) {
  DS_REQUIRE(d != nullptr, "null descriptor");
  DS_REQUIRE(d->dtype == DS_BF16 || d->dtype == DS_FP16 || d->dtype == DS_FP32, "KV caches must use BF16, FP16 or FP32");
  DS_REQUIRE(d->rows >= 0, "row counts must be non-negative");
  DS_REQUIRE(d->num_kv_heads > 0 && d->head_dim > 0, "head counts and sizes must be positive");
  const int size = d->dtype == DS_FP32 ? 4 : 2;
  DS_SUPPORTED(static_cast<int64_t>(d->head_dim) * size % 16 == 0, "heads must be multiples of 16 bytes");
  DS_SUPPORTED(d->rows <= kMaxRows, "at most %d rows", kMaxRows);
  DS_REQUIRE(d->block_size > 0 && d->num_blocks > 0 && d->max_blocks > 0, "block sizes and counts must be positive");
  DS_SUPPORTED(d->block_size <= (1 << 30), "at most 2^30 tokens per page");  // a row's pages are counted in 32 bits
  DS_REQUIRE(d->capacity > 0, "capacity must be positive");
  DS_REQUIRE(d->sinks >= 0 && d->recent >= 0, "sinks and recent must not be negative");
  DS_SUPPORTED(static_cast<int64_t>(d->sinks) + d->recent <= (1 << 29), "at most 2^29 tokens that are always kept");
  if (d->rows == 0) return clear_error();
  DS_REQUIRE(d->key_cache && d->value_cache && d->mass && d->positions && d->settled && d->block_table && d->target_len &&
                 d->keep_len && d->kept_len,
             "null tensor pointer");
  // Heads of a row read its lengths while one of them writes its new one.
  const auto apart = [&](const int32_t* x) {
    const uintptr_t one = reinterpret_cast<uintptr_t>(d->kept_len), other = reinterpret_cast<uintptr_t>(x);
    const uintptr_t bytes = sizeof(int32_t) * static_cast<uintptr_t>(d->rows);
    return one + bytes <= other || other + bytes <= one;
  };
  DS_REQUIRE(apart(d->target_len) && apart(d->keep_len), "kept_len must be memory of its own");
  const int64_t strides[] = {d->k_block_stride, d->k_token_stride, d->k_head_stride,
                             d->v_block_stride, d->v_token_stride, d->v_head_stride};
  for (int64_t s : strides) DS_REQUIRE(s >= 0 && s * size % 16 == 0, "page and head strides must be multiples of 16 bytes");
  DS_REQUIRE(aligned(d->key_cache) && aligned(d->value_cache), "KV caches must be 16-byte aligned");
  const int64_t capacity = std::min<int64_t>(static_cast<int64_t>(d->max_blocks) * d->block_size, d->capacity);
  DS_SUPPORTED(capacity <= (1 << 29), "rows of at most 2^29 keys");
  DS_SUPPORTED(static_cast<int64_t>(d->rows) * d->num_kv_heads <= 65535, "at most 65535 heads of all rows");
  DS_REQUIRE(d->workspace && d->workspace_bytes >= evict_workspace_bytes(d->rows, d->num_kv_heads, static_cast<int>(capacity)) &&
                 (reinterpret_cast<uintptr_t>(d->workspace) & 255u) == 0,
             "workspace must be 256-byte aligned and hold ds_evict_workspace_bytes()");
  EvictArgs a{};
  a.k = static_cast<char*>(d->key_cache);
  a.k_block = size * d->k_block_stride, a.k_token = size * d->k_token_stride, a.k_head = size * d->k_head_stride;
  a.v = static_cast<char*>(d->value_cache);
  a.v_block = size * d->v_block_stride, a.v_token = size * d->v_token_stride, a.v_head = size * d->v_head_stride;
  a.mass = d->mass;
  a.m_row = d->mass_row_stride, a.m_head = d->mass_head_stride;
  a.positions = d->positions;
  a.p_row = d->positions_row_stride, a.p_head = d->positions_head_stride;
  a.settled = d->settled;
  a.table = d->block_table;
  a.bt_stride = d->bt_stride;
  a.ref_counts = d->ref_counts;
  a.t_len = d->target_len, a.keep_len = d->keep_len, a.kept_len = d->kept_len;
  a.capacity = static_cast<int>(capacity);
  a.num_blocks = d->num_blocks;
  a.block_size = d->block_size;
  a.rows = d->rows, a.hkv = d->num_kv_heads, a.pieces = d->head_dim * size / 16;
  a.sinks = d->sinks, a.recent = d->recent;
  a.groups = static_cast<int>((capacity + 63) / 64);
  const int heads = d->rows * d->num_kv_heads;
  a.heads = static_cast<Head*>(d->workspace);
  a.lists = reinterpret_cast<Group*>(static_cast<char*>(d->workspace) + rounded(heads * sizeof(Head)));
  a.status = d->status;
  if (capacity <= 4096) evict_select_kernel<4096><<<heads, kSelectThreads, 0, stream>>>(a);
  else if (capacity <= 8192) evict_select_kernel<8192><<<heads, kSelectThreads, 0, stream>>>(a);
  else evict_select_kernel<32768><<<heads, kSelectThreads, 0, stream>>>(a);
  // Workgroups of a head: enough for all its moves at most, and to fill the chip a few times over.
  const int64_t full = (capacity / 2 + kMoves) / kMoves, fill = std::max<int64_t>(1, 16LL * device_cu_count() / heads);
  evict_move_kernel<<<dim3(static_cast<int>(std::min(full, fill)), heads), kMoveThreads, 0, stream>>>(a);
  return check_launch("ds_evict");
}

}  // namespace
}  // namespace ds355

extern "C" size_t ds_evict_workspace_bytes(int rows, int num_kv_heads, int capacity) {
  return ds355::evict_workspace_bytes(rows, num_kv_heads, capacity);
}

extern "C" int ds_evict(ds_stream_t stream, const ds_evict_desc* desc) {
  return ds355::evict_impl(reinterpret_cast<hipStream_t>(stream), desc);
}

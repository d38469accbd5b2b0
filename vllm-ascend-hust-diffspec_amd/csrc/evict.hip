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
// evict_select_kernel: a workgroup a (row, KV head).  The k-th largest value is found byte by byte from
// histograms of an order-preserving integer; the moves go to a list, and the masses and positions with
// them.  evict_move_kernel moves the keys and values.
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
  int most;           // moves of a head, at most
  int32_t* counts;    // [rows * hkv], -1: the row is left alone
  int2* moves;        // [rows * hkv][most]: source, destination
  int32_t* status;
};

// Unsigned integers in the order of floating-point values; NaN below all.
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 0;
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One head's slots.
struct Slots {
  const float* mass;
  const int32_t* positions;
  int known, gone, sinks, newest;  // tokens at or past `newest` are always kept
  __device__ __forceinline__ int position(int t) const { return t < known ? positions[t] : t + gone; }
  __device__ __forceinline__ uint32_t value(int t) const {
    const int p = position(t);
    return p < sinks || p >= newest ? 0xffffffffu : ordered(mass[t]);
  }
};

__device__ __forceinline__ void report(const EvictArgs& a, uint32_t bits) {
  if (a.status) __hip_atomic_fetch_or(a.status, static_cast<int>(bits), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Exclusive prefix over the waves of a count that is the same in a wave's lanes; `total` gets the sum.
__device__ __forceinline__ int wave_prefix(int count, int* scratch, int& total) {
  const int wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[wave] = count;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < kSelectWaves; ++w) {
    if (w < wave) before += scratch[w];
    total += scratch[w];
  }
  return before;
}

__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(EvictArgs a) {
  __shared__ int histogram[256];
  __shared__ int scratch[kSelectWaves];
  __shared__ int found, left, refused;
  const int b = blockIdx.x / a.hkv, h = blockIdx.x - b * a.hkv;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int n = a.t_len[b], keep = a.keep_len[b];
  uint32_t bits = 0;
  if (n > a.capacity) {
    bits = kStatusLength;
  } else if (n > 0 && (keep < 0 || (keep < n && a.sinks > keep - a.recent))) {
    bits = kStatusBudget;
  }
  if (tid == 0) refused = 0;
  __syncthreads();
  if (!bits && n > keep && n > 0) {
    for (int i = tid; i < ceil_div(n, a.block_size); i += kSelectThreads) {
      const int page = a.table[b * a.bt_stride + i];
      if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.num_blocks)) {
        atomicOr(&refused, kStatusPage);
      } else if (a.ref_counts && i * a.block_size < keep && a.ref_counts[page] > 1) {
        atomicOr(&refused, kStatusShared);
      }
    }
  }
  __syncthreads();
  bits |= refused;
  const bool work = !bits && n > keep && n > 0;
  if (tid == 0) {
    if (h == 0) a.kept_len[b] = work ? keep : max(n, 0);
    if (!work) a.counts[blockIdx.x] = -1;
    if (bits && h == 0) report(a, bits);
  }
  if (!work) return;
  float* mass = a.mass + b * a.m_row + h * a.m_head;
  int32_t* positions = a.positions + b * a.p_row + h * a.p_head;
  const int known = min(max(a.settled[2 * b], 0), n), gone = a.settled[2 * b + 1];
  const Slots slots{mass, positions, known, gone, a.sinks, n + gone - a.recent};

  // The keep-th largest value, byte by byte, and how many of its equals are kept.
  uint32_t value = 0;
  int need = keep;  // kept values among those that share the bytes found so far
  for (int shift = 24; shift >= 0 && need > 0; shift -= 8) {
    for (int i = tid; i < 256; i += kSelectThreads) histogram[i] = 0;
    __syncthreads();
    for (int t = tid; t < n; t += kSelectThreads) {
      const uint32_t x = slots.value(t);
      if (shift == 24 || (x >> (shift + 8)) == (value >> (shift + 8))) atomicAdd(&histogram[(x >> shift) & 255], 1);
    }
    __syncthreads();
    if (wave == 0) {  // bins from the largest down, four a lane
      int own[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        own[i] = histogram[255 - 4 * lane - i];
        sum += own[i];
      }
      int above = wave_inclusive_scan(sum) - sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (above < need && need <= above + own[i]) {
          found = 255 - 4 * lane - i;
          left = need - above;
        }
        above += own[i];
      }
    }
    __syncthreads();
    value |= static_cast<uint32_t>(found) << shift;
    need = left;
    __syncthreads();
  }

  // Slots in order: a wave takes a range of them, 64 at a time.
  const int span = ceil_div(ceil_div(n, kSelectWaves), 64) * 64;
  const int begin = min(wave * span, n), end = min(begin + span, n);
  const uint64_t below = (1ull << lane) - 1;
  int total;
  int ties = 0;
  for (int t = begin + lane; t - lane < end; t += 64) ties += __popcll(__ballot(t < end && slots.value(t) == value));
  const int ties_before = wave_prefix(ties, scratch, total);
  auto keeps = [&](int t, int& tie) {  // whether slot t is kept; counts the equals
    const uint32_t x = t < end ? slots.value(t) : 0;
    const uint64_t equal = __ballot(t < end && x == value);
    const bool kept = t < end && keep > 0 && (x > value || (x == value && tie + __popcll(equal & below) < need));
    tie += __popcll(equal);
    return kept;
  };
  int holes = 0, movers = 0, tie = ties_before;
  for (int t = begin + lane; t - lane < end; t += 64) {
    const bool kept = keeps(t, tie);
    holes += __popcll(__ballot(t < end && t < keep && !kept));
    movers += __popcll(__ballot(kept && t >= keep));
  }
  int hole = wave_prefix(holes, scratch, total);
  const int count = total;  // as many movers as holes
  int mover = wave_prefix(movers, scratch, total);
  int2* moves = a.moves + static_cast<int64_t>(blockIdx.x) * a.most;
  tie = ties_before;
  for (int t = begin + lane; t - lane < end; t += 64) {
    const bool kept = keeps(t, tie);
    const uint64_t to = __ballot(t < end && t < keep && !kept), from = __ballot(kept && t >= keep);
    if ((to >> lane) & 1) moves[hole + __popcll(to & below)].y = t;
    if ((from >> lane) & 1) moves[mover + __popcll(from & below)].x = t;
    if (kept && t < keep && t >= known) positions[t] = t + gone;
    hole += __popcll(to);
    mover += __popcll(from);
  }
  __syncthreads();
  for (int i = tid; i < count; i += kSelectThreads) {
    const int2 move = moves[i];
    positions[move.y] = slots.position(move.x);
    mass[move.y] = mass[move.x];
  }
  __syncthreads();
  for (int t = keep + tid; t < n; t += kSelectThreads) mass[t] = 0.f;
  if (tid == 0) a.counts[blockIdx.x] = count;
}

__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a) {
  const int count = a.counts[blockIdx.y];
  if (count < 0) return;
  const int b = blockIdx.y / a.hkv, h = blockIdx.y - b * a.hkv;
  if (h == 0 && blockIdx.x == 0 && threadIdx.x == 0) {
    a.settled[2 * b + 1] += a.t_len[b] - a.keep_len[b];
    a.settled[2 * b] = a.keep_len[b];
  }
  const int32_t* pages = a.table + b * a.bt_stride;
  const int2* moves = a.moves + static_cast<int64_t>(blockIdx.y) * a.most;
  const int64_t total = static_cast<int64_t>(count) * a.pieces;
  for (int64_t i = blockIdx.x * kMoveThreads + threadIdx.x; i < total; i += gridDim.x * kMoveThreads) {
    const int move = static_cast<int>(i / a.pieces), piece = static_cast<int>(i - static_cast<int64_t>(move) * a.pieces);
    const int2 m = moves[move];
    const int from = m.x / a.block_size, to = m.y / a.block_size;
    const int64_t source = pages[from], target = pages[to];
    const int in_from = m.x - from * a.block_size, in_to = m.y - to * a.block_size;
    *reinterpret_cast<u32x4*>(a.k + target * a.k_block + in_to * a.k_token + h * a.k_head + 16 * piece) =
        *reinterpret_cast<const u32x4*>(a.k + source * a.k_block + in_from * a.k_token + h * a.k_head + 16 * piece);
    *reinterpret_cast<u32x4*>(a.v + target * a.v_block + in_to * a.v_token + h * a.v_head + 16 * piece) =
        *reinterpret_cast<const u32x4*>(a.v + source * a.v_block + in_from * a.v_token + h * a.v_head + 16 * piece);
  }
}

size_t rounded(size_t n) { return (n + 255) & ~size_t{255}; }

size_t evict_workspace_bytes(int rows, int num_kv_heads, int capacity) {
  if (rows <= 0 || num_kv_heads <= 0 || capacity <= 0) return 0;
  const size_t heads = static_cast<size_t>(rows) * num_kv_heads;
  return rounded(heads * sizeof(int32_t)) + heads * (capacity / 2 + 1) * sizeof(int2);
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
  DS_REQUIRE(d->capacity > 0, "capacity must be positive");
  DS_REQUIRE(d->sinks >= 0 && d->recent >= 0, "sinks and recent must not be negative");
  DS_SUPPORTED(static_cast<int64_t>(d->sinks) + d->recent <= (1 << 29), "at most 2^29 tokens that are always kept");
  if (d->rows == 0) return clear_error();
  DS_REQUIRE(d->key_cache && d->value_cache && d->mass && d->positions && d->settled && d->block_table && d->target_len &&
                 d->keep_len && d->kept_len,
             "null tensor pointer");
  // Heads of a row read its lengths while one of them writes its new one.
  DS_REQUIRE(d->kept_len != d->target_len && d->kept_len != d->keep_len, "kept_len must be memory of its own");
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
  a.most = static_cast<int>(capacity / 2 + 1);
  const int heads = d->rows * d->num_kv_heads;
  a.counts = static_cast<int32_t*>(d->workspace);
  a.moves = reinterpret_cast<int2*>(static_cast<char*>(d->workspace) + rounded(heads * sizeof(int32_t)));
  a.status = d->status;
  evict_select_kernel<<<heads, kSelectThreads, 0, stream>>>(a);
  // Workgroups of a head: enough for all its moves at most, and to fill the chip a few times over.
  const int64_t full = (static_cast<int64_t>(a.most) * a.pieces + kMoveThreads - 1) / kMoveThreads;
  const int64_t fill = std::max<int64_t>(1, 16LL * device_cu_count() / heads);
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

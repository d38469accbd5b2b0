// The attention weight that each cached key receives from a step's query tokens.
//
// What an eviction goes by: with the rows, pages and causal ends (and windows) of the chunk attention and
// the LSE that it wrote,
//
//   mass[b, h, t] = decay previous[b, h, t] + sum over the query tokens i of row b that see key t, and
//                   the query heads g of KV head h, of exp(scale q_ig . k_t - lse_ig).
//
// The probabilities are those of the attention, so the keys are read once more, and the values not at all.
// A wave holds 64 keys (32 of 256 dimensions) in registers as the columns of the score product, and the
// query rows (row = token * group + head in the group) go by in shared memory, 64 at a time.  A lane's
// results are then 16 query rows of its own key, and the sum over the rows is the lane's own.  Tiles of
// keys with many query rows are cut into parts of the rows, whose sums mass_join_kernel adds up in order.
#include <cmath>

#include "matrix.h"

namespace ds355 {
namespace {

constexpr int kQueryRows = 64;  // staged query rows
constexpr int kMinPart = 4;     // staged tiles below which the query rows are not cut
constexpr int kPartsPerSlot = 4;
constexpr uint32_t kStatusRow = 1;     // a row's query tokens are out of range
constexpr uint32_t kStatusLength = 2;  // a row is longer than its block table or its mass
constexpr uint32_t kStatusPage = 4;    // a page id is out of range

constexpr int kWaves = 4;
constexpr int wave_keys(int d) { return d <= 128 ? 64 : 32; }
constexpr int mass_tile(int d) { return kWaves * wave_keys(d); }
constexpr int kMostKeys = 256;  // keys of a tile, at most
int mass_slots() { return 2 * device_cu_count(); }  // workgroups that run at a time

template <int D>
struct Mass {
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kTile = mass_tile(D);
  static constexpr int kColumns = wave_keys(D) / 32;  // blocks of 32 keys of a wave
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kPieces = D / 8;
  static constexpr int kSteps = D / 16;
};

struct MassArgs {
  const uint16_t* q;
  int64_t q_row, q_head;
  const char* k;
  int64_t k_block, k_token, k_head;  // bytes
  const float* lse;
  int64_t l_row, l_head;
  const float* previous;
  int64_t p_row, p_head;
  float* mass;
  int64_t m_row, m_head;
  const int32_t* table;
  int64_t bt_stride;
  int capacity;  // keys that a row can hold
  int num_blocks, block_size;
  const int32_t* q_start;
  const int32_t* q_len;
  const int32_t* t_len;
  int rows, tokens, hkv, group, window;
  int tile;  // keys of a tile
  int slots;
  float scale_log2;  // |scale| log2 e
  uint32_t q_sign;   // sign bits that a negative scale turns in the queries
  float decay;
  float* partial;  // [parts of cut tiles][KV head][kMostKeys]
  int32_t* status;
};

// ---------------------------------------------------------------------------------------------
// The layout of the work, derived by every workgroup from the lengths.
// ---------------------------------------------------------------------------------------------
struct Row {
  int start, len, keys;
};
__device__ __forceinline__ Row row_of(const MassArgs& a, int b, bool report) {
  Row r{a.q_start[b], a.q_len[b], a.t_len[b]};
  uint32_t bits = 0;
  if (r.len <= 0) {
    r.len = 0;
  } else if (r.start < 0 || r.len > a.tokens || r.start > a.tokens - r.len) {
    r.len = 0;
    bits |= kStatusRow;
  }
  if (r.keys > a.capacity) bits |= kStatusLength;
  if (bits && report && a.status) {
    __hip_atomic_fetch_or(a.status, static_cast<int>(bits), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  r.keys = r.len ? min(max(r.keys, 0), a.capacity) : 0;
  return r;
}

struct Layout {
  int first[kMaxRows + 1];  // parts of the rows before, of one KV head
  int cut[kMaxRows + 1];    // those of them that are one of several of a tile
  int cap;                  // staged tiles of a part, at most
};

// Parts of each tile of the row.
__device__ __forceinline__ int row_parts(const MassArgs& a, int len, int cap) {
  return max(ceil_div(ceil_div(len * a.group, kQueryRows), cap), 1);
}

__device__ __forceinline__ void make_layout(const MassArgs& a, Layout& y, bool report) {
  __shared__ int scratch[4];
  __shared__ unsigned long long work;
  if (threadIdx.x == 0) work = 0;
  __syncthreads();
  unsigned long long mine = 0;
  for (int b = threadIdx.x; b < a.rows; b += blockDim.x) {
    const Row r = row_of(a, b, report);
    mine += static_cast<unsigned long long>(ceil_div(r.keys, a.tile)) * ceil_div(r.len * a.group, kQueryRows);
  }
  if (mine) atomicAdd(&work, mine);
  __syncthreads();
  const unsigned long long most = static_cast<unsigned long long>(kPartsPerSlot) * a.slots;
  const unsigned long long share = (work * a.hkv + most - 1) / most;
  const int cap = static_cast<int>(min(max(share, static_cast<unsigned long long>(kMinPart)), 1ull << 25));
  if (threadIdx.x == 0) y.cap = cap;
  build_row_prefix(a.rows, y.first, scratch, [&](int b) {
    const Row r = row_of(a, b, false);
    return ceil_div(r.keys, a.tile) * row_parts(a, r.len, cap);
  });
  build_row_prefix(a.rows, y.cut, scratch, [&](int b) {
    const Row r = row_of(a, b, false);
    const int parts = row_parts(a, r.len, cap);
    return parts > 1 ? ceil_div(r.keys, a.tile) * parts : 0;
  });
}

// One part: a tile of a row's keys, and which of its query rows.
struct Part {
  int row, start, len, keys, seen;
  int tile, part, parts, slot;
};
__device__ __forceinline__ Part part_at(const MassArgs& a, const Layout& y, int i) {
  Part p;
  p.row = uniform(find_row(y.first, a.rows, i));
  const Row r = row_of(a, p.row, false);
  p.start = uniform(r.start), p.len = uniform(r.len), p.keys = uniform(r.keys);
  p.seen = p.keys - p.len;
  p.parts = row_parts(a, p.len, uniform(y.cap));
  const int in_row = i - uniform(y.first[p.row]);
  p.tile = in_row / p.parts;
  p.part = in_row - p.tile * p.parts;
  p.slot = uniform(y.cut[p.row]) + in_row;
  return p;
}

// Query rows that see key t: [from, to) (rows hold at most 2^29 keys, and windows count as no more).
__device__ __forceinline__ int first_row(const MassArgs& a, const Part& p, int t) {
  return min(max(t - p.seen, 0), p.len) * a.group;
}
__device__ __forceinline__ int end_row(const MassArgs& a, const Part& p, int t) {
  return min(max(t - p.seen + a.window, 0), p.len) * a.group;
}

template <int D>
__device__ __forceinline__ int row_turn(int t) {
  return D == 64 ? (t >> 1) & 7 : t & 15;
}

template <int DT, int D>
__global__ __launch_bounds__(Mass<D>::kThreads, 2) void attention_mass_kernel(MassArgs a) {
  using M = Mass<D>;
  __shared__ Layout layout;
  __shared__ __attribute__((aligned(512))) char lds[kQueryRows * M::kRowBytes];
  __shared__ __attribute__((aligned(16))) float lse[kQueryRows];
  make_layout(a, layout, blockIdx.x == 0);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), half = lane >> 5;
  const int total = uniform(layout.first[a.rows]) * a.hkv;
  for (int i = blockIdx.x; i < total; i += gridDim.x) {
    const int entry = i / a.hkv, h = i - entry * a.hkv;
    const Part p = part_at(a, layout, entry);
    const int t0 = p.tile * M::kTile + wave * 32 * M::kColumns;
    u32x4 k[M::kColumns][M::kSteps];
    int from[M::kColumns], to[M::kColumns];
#pragma unroll
    for (int c = 0; c < M::kColumns; ++c) {
      const int t = t0 + 32 * c + (lane & 31);
      from[c] = first_row(a, p, t), to[c] = t < p.keys ? end_row(a, p, t) : 0;
      const int n = min(t, p.keys - 1), index = n / a.block_size, in = n - index * a.block_size;
      const int page = a.table[p.row * a.bt_stride + index];
      const bool fine = static_cast<unsigned>(page) < static_cast<unsigned>(a.num_blocks);
      if (!fine && a.status) {
        __hip_atomic_fetch_or(a.status, static_cast<int>(kStatusPage), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      const char* src = a.k + (fine ? page : 0) * a.k_block + in * a.k_token + h * a.k_head + 16 * half;
#pragma unroll
      for (int s = 0; s < M::kSteps; ++s) {
        k[c][s] = *reinterpret_cast<const u32x4*>(src + 32 * s);
        if (!fine) k[c][s] = u32x4{0, 0, 0, 0};
      }
    }
    // The staged tiles of query rows that see some key of the tile, and the part's share of them.
    const int last_key = min((p.tile + 1) * M::kTile, p.keys) - 1;
    const int lo = first_row(a, p, p.tile * M::kTile) / kQueryRows, hi = ceil_div(end_row(a, p, last_key), kQueryRows);
    const int n = max(hi - lo, 0);
    const int begin = lo + static_cast<int>(static_cast<int64_t>(n) * p.part / p.parts);
    const int end = lo + static_cast<int>(static_cast<int64_t>(n) * (p.part + 1) / p.parts);
    const int rows = p.len * a.group;
    float sum[M::kColumns];
#pragma unroll
    for (int c = 0; c < M::kColumns; ++c) sum[c] = 0.f;
    for (int block = begin; block < end; ++block) {
      __syncthreads();
      for (int j = threadIdx.x; j < kQueryRows * M::kPieces; j += M::kThreads) {
        const int row = j / M::kPieces, c = j % M::kPieces, r = min(block * kQueryRows + row, rows - 1);
        const int token = p.start + r / a.group, head = h * a.group + r % a.group;
        *reinterpret_cast<u32x4*>(lds + row * M::kRowBytes + 16 * (c ^ row_turn<D>(row))) =
            *reinterpret_cast<const u32x4*>(a.q + token * a.q_row + head * a.q_head + 8 * c) ^ a.q_sign;
      }
      if (threadIdx.x < kQueryRows) {
        const int r = min(block * kQueryRows + static_cast<int>(threadIdx.x), rows - 1);
        const float x = a.lse[(p.start + r / a.group) * a.l_row + (h * a.group + r % a.group) * a.l_head];
        // A query head that saw nothing adds nothing.
        lse[threadIdx.x] = x == -INFINITY ? INFINITY : x * kLog2eP;
      }
      __syncthreads();
#pragma unroll
      for (int b = 0; b < kQueryRows / 32; ++b) {
        const int r0 = block * kQueryRows + 32 * b;
        f32x16 sc[M::kColumns];
#pragma unroll
        for (int c = 0; c < M::kColumns; ++c) {
#pragma unroll
          for (int e = 0; e < 16; ++e) sc[c][e] = 0.f;
        }
        const int row = 32 * b + (lane & 31);
#pragma unroll
        for (int s = 0; s < M::kSteps; ++s) {
          const u32x4 q = *reinterpret_cast<const u32x4*>(lds + row * M::kRowBytes + 16 * ((2 * s + half) ^ row_turn<D>(row)));
#pragma unroll
          for (int c = 0; c < M::kColumns; ++c) sc[c] = mfma32<DT>(q, k[c][s], sc[c]);
        }
        f32x4 x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = *reinterpret_cast<const f32x4*>(lse + 32 * b + 8 * e + 4 * half);
#pragma unroll
        for (int c = 0; c < M::kColumns; ++c) {
          const bool whole = __all(from[c] <= r0 && r0 + 32 <= to[c]);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[c][e], a.scale_log2, -x[e >> 2][e & 3]));
            const int r = r0 + 8 * (e >> 2) + 4 * half + (e & 3);
            if (whole) sum[c] += w;
            else sum[c] += r >= from[c] && r < to[c] ? w : 0.f;
          }
        }
      }
    }
#pragma unroll
    for (int c = 0; c < M::kColumns; ++c) {
      sum[c] += other_half(sum[c]);
      const int t = t0 + 32 * c + lane;
      if (half || t >= p.keys) continue;
      if (p.parts > 1) {
        a.partial[(static_cast<int64_t>(p.slot) * a.hkv + h) * kMostKeys + t - p.tile * M::kTile] = sum[c];
      } else {
        const float old = a.previous ? a.decay * a.previous[p.row * a.p_row + h * a.p_head + t] : 0.f;
        a.mass[p.row * a.m_row + h * a.m_head + t] = old + sum[c];
      }
    }
  }
}

// Adds up the parts of cut tiles, a thread a key.
__global__ __launch_bounds__(kMostKeys) void mass_join_kernel(MassArgs a) {
  __shared__ Layout layout;
  make_layout(a, layout, false);
  const int total = uniform(layout.cut[a.rows]) * a.hkv;
  for (int i = blockIdx.x; i < total; i += gridDim.x) {
    const int entry = i / a.hkv, h = i - entry * a.hkv;
    // The rows without cut tiles have no entries here.
    const int row = uniform(find_row(layout.cut, a.rows, entry));
    const int in_row = entry - uniform(layout.cut[row]);
    const Part p = part_at(a, layout, uniform(layout.first[row]) + in_row);
    if (p.part) continue;
    const int t = p.tile * a.tile + threadIdx.x;
    if (static_cast<int>(threadIdx.x) >= a.tile || t >= p.keys) continue;
    float sum = a.previous ? a.decay * a.previous[p.row * a.p_row + h * a.p_head + t] : 0.f;
    for (int j = 0; j < p.parts; ++j) {
      sum += a.partial[(static_cast<int64_t>(p.slot + j) * a.hkv + h) * kMostKeys + threadIdx.x];
    }
    a.mass[p.row * a.m_row + h * a.m_head + t] = sum;
  }
}

// Parts of cut tiles: a row's tiles have at most twice the parts that their staged tiles fill, so at most
// 2 kPartsPerSlot for each workgroup that runs at a time, all KV heads together.
int64_t partial_parts() { return 2LL * kPartsPerSlot * mass_slots() + 1; }
size_t mass_workspace_bytes() { return static_cast<size_t>(partial_parts()) * kMostKeys * sizeof(float); }

template <int DT>
void launch_dim(hipStream_t stream, int d, const MassArgs& a) {
  if (d == 64) attention_mass_kernel<DT, 64><<<a.slots, Mass<64>::kThreads, 0, stream>>>(a);
  else if (d == 128) attention_mass_kernel<DT, 128><<<a.slots, Mass<128>::kThreads, 0, stream>>>(a);
  else attention_mass_kernel<DT, 256><<<a.slots, Mass<256>::kThreads, 0, stream>>>(a);
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int attention_mass_impl(hipStream_t stream, const ds_attention_mass_desc* d) {
  DS_REQUIRE(d != nullptr, "null descriptor");
  DS_REQUIRE(d->dtype == DS_BF16 || d->dtype == DS_FP16, "queries and key cache must use BF16 or FP16");
  DS_REQUIRE(d->rows >= 0 && d->tokens >= 0, "row and token counts must be non-negative");
  DS_REQUIRE(d->num_q_heads > 0 && d->num_kv_heads > 0 && d->num_q_heads % d->num_kv_heads == 0,
             "query heads must be divisible by KV heads");
  DS_SUPPORTED(d->head_dim == 64 || d->head_dim == 128 || d->head_dim == 256, "head_dim must be 64, 128 or 256");
  DS_SUPPORTED(d->rows <= kMaxRows, "at most %d rows", kMaxRows);
  DS_REQUIRE(d->block_size > 0 && d->num_blocks > 0 && d->max_blocks > 0, "block sizes and counts must be positive");
  DS_REQUIRE(d->capacity > 0, "capacity must be positive");
  DS_REQUIRE(d->window >= 0, "window must not be negative (0: no window)");
  DS_SUPPORTED(d->block_size <= (1 << 20), "at most 2^20 tokens per page");
  if (d->rows == 0 || d->tokens == 0) return clear_error();
  DS_REQUIRE(d->query && d->key_cache && d->lse && d->mass && d->block_table && d->query_start && d->query_len &&
                 d->target_len,
             "null tensor pointer");
  const int64_t strides[] = {d->q_row_stride, d->q_head_stride, d->k_block_stride, d->k_token_stride, d->k_head_stride};
  for (int64_t s : strides) DS_REQUIRE(s >= 0 && s % 8 == 0, "row, page and head strides must be multiples of 8 elements");
  for (int i = 2; i < 5; ++i) DS_SUPPORTED(strides[i] < (1 << 30), "pages of at most 2^30 elements");
  DS_SUPPORTED(d->block_size * d->k_token_stride + d->num_kv_heads * d->k_head_stride < (1 << 30),
               "pages of at most 2^30 elements");
  DS_REQUIRE(aligned(d->query) && aligned(d->key_cache), "query and key cache must be 16-byte aligned");
  DS_REQUIRE(d->workspace && d->workspace_bytes >= mass_workspace_bytes() &&
                 (reinterpret_cast<uintptr_t>(d->workspace) & 255u) == 0,
             "workspace must be 256-byte aligned and hold ds_attention_mass_workspace_bytes()");
  const int group = d->num_q_heads / d->num_kv_heads;
  const int64_t capacity = std::min<int64_t>(static_cast<int64_t>(d->max_blocks) * d->block_size, d->capacity);
  const int tile = mass_tile(d->head_dim);
  DS_SUPPORTED(capacity <= (1 << 29), "rows of at most 2^29 keys");
  DS_SUPPORTED(d->tokens <= (1 << 20), "at most 2^20 query tokens");
  // Parts are counted in 32 bits.
  const int64_t tiles = static_cast<int64_t>(d->rows) * ((capacity + tile - 1) / tile);
  DS_SUPPORTED(static_cast<int64_t>(d->tokens) * group < (1 << 30) && tiles * d->num_kv_heads + partial_parts() < (1 << 30),
               "too many query tokens, KV heads or keys for one launch");
  MassArgs a{};
  a.q = static_cast<const uint16_t*>(d->query);
  a.q_row = d->q_row_stride, a.q_head = d->q_head_stride;
  a.k = static_cast<const char*>(d->key_cache);
  a.k_block = 2 * d->k_block_stride, a.k_token = 2 * d->k_token_stride, a.k_head = 2 * d->k_head_stride;
  a.lse = d->lse;
  a.l_row = d->lse_token_stride, a.l_head = d->lse_head_stride;
  a.previous = d->previous;
  a.p_row = d->previous_row_stride, a.p_head = d->previous_head_stride;
  a.mass = d->mass;
  a.m_row = d->mass_row_stride, a.m_head = d->mass_head_stride;
  a.table = d->block_table;
  a.bt_stride = d->bt_stride;
  a.capacity = static_cast<int>(capacity);
  a.num_blocks = d->num_blocks;
  a.block_size = d->block_size;
  a.q_start = d->query_start, a.q_len = d->query_len, a.t_len = d->target_len;
  a.rows = d->rows, a.tokens = d->tokens, a.hkv = d->num_kv_heads, a.group = group;
  a.window = d->window ? std::min(d->window, 1 << 29) : 1 << 29;
  a.tile = tile;
  a.slots = mass_slots();
  a.scale_log2 = std::fabs(d->scale) * kLog2eP;
  a.q_sign = d->scale < 0.f ? 0x80008000u : 0u;
  a.decay = d->decay;
  a.partial = static_cast<float*>(d->workspace);
  a.status = d->status;
  if (d->dtype == DS_BF16) launch_dim<DS_BF16>(stream, d->head_dim, a);
  else launch_dim<DS_FP16>(stream, d->head_dim, a);
  // Fewer query rows than a part's make no parts.
  if (static_cast<int64_t>(d->tokens) * group > kMinPart * kQueryRows) {
    mass_join_kernel<<<a.slots, kMostKeys, 0, stream>>>(a);
  }
  return check_launch("ds_attention_mass");
}

}  // namespace
}  // namespace ds355

extern "C" size_t ds_attention_mass_workspace_bytes(void) { return ds355::mass_workspace_bytes(); }

extern "C" int ds_attention_mass(ds_stream_t stream, const ds_attention_mass_desc* desc) {
  return ds355::attention_mass_impl(reinterpret_cast<hipStream_t>(stream), desc);
}

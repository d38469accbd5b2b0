// The attention weight that each cached key receives from a step's query tokens.
//
// What an eviction goes by: with the rows, pages and causal ends (and windows) of the chunk attention and
// the LSE that it wrote,
//
//   mass[b, h, t] = decay previous[b, h, t] + sum over the query tokens i of row b that see key t, and
//                   the query heads g of KV head h, of exp(scale q_ig . k_t - lse_ig).
//
// The probabilities are those of the attention, so the keys are read once more, and the values not at all.
// A wave holds 32 keys in registers as the columns of the score product, and the query rows (row = token *
// group + head in the group) go by in shared memory, 64 at a time.  A lane's results are then 16 query rows
// of its own key, and the sum over the rows is the lane's own.  Tiles of keys with many query rows are cut
// into parts of the rows, whose sums mass_join_kernel adds up in order.
//
// What bounds it: with few query rows the keys' bytes (16 tokens, 32 heads on 4 of 128 dimensions, over 4 k to 16 k keys:
// 43 us, 3.9 TB/s); with many vector issue (52% of the cycles at 128 dimensions, 62% at 64, the exponentials 30% of that)
// and what a part costs beside its blocks (2048 tokens on 8 k keys, 32 heads on 8: 169 us, 711 TFLOP/s; 6 times 32 tokens,
// 64 heads on 8 of 64 dimensions, whose parts are of four blocks, 50 us).
#include <cmath>

#include "matrix.h"

namespace ds355 {
namespace {

// Staged query rows, a block: 64, whose two products and weighings overlap, or 32 where the rows have about as
// many, so that more workgroups fit a CU.  16 rows of 8 query rows each over 4 k to 16 k keys take 43 us with 32
// and 53 with 64, 6 rows of 256 take 64 and 50, one of 8192 takes 176 and 170.
constexpr int kMostRows = 64;
// Query rows below which they are not cut: 128 tokens on 1 k keys, 32 heads on 4 of 128 dimensions, take 17.7 us with 256, 15.7
// with 128 and 23.5 with 512, 100 rows of 8 tokens beside one of 1500 147, 157 and 147.
constexpr int kMinPart = 256;
// What a slot's workgroup gets of the least parts.  More are dealt more evenly and cost more: 40 rows of 64 tokens on 2 k keys take
// 95 us with 8, 88 with 4 and 95 with 16, 65 such rows 135, 134 and 188, 16 rows on 4 k 79, 77 and 78.
constexpr int kPartsPerSlot = 8;
// Rows up to which the sizes of parts are compared, since a lane goes over all rows: 16 rows of 64 tokens on 4 k keys take
// 79 us, and 100 uncompared; 65 rows of 64 on 2 k 135 either way, 100 rows of 8 beside one of 1500 147, and 169 compared.
constexpr int kComparedRows = 64;
constexpr uint32_t kStatusRow = 1;     // a row's query tokens are out of range
constexpr uint32_t kStatusLength = 2;  // a row is longer than its block table or its mass
constexpr uint32_t kStatusPage = 4;    // a page id is out of range

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kTile = 32 * kWaves;  // keys of a workgroup
// Workgroups of a CU.
constexpr int mass_groups(int d, int block) { return d == 64 ? 4 : d == 256 ? 1 : block == 64 ? 2 : 3; }
constexpr int kMostGroups = 4;

template <int D, int R>
struct Mass {
  static constexpr int kQueryRows = R;
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kPieces = D / 8;
  static constexpr int kSteps = D / 16;
  static constexpr int kPerLoad = 64 / kPieces;                      // keys or rows that one load of a wave covers
  static constexpr int kKeyLoads = 32 / kPerLoad;                    // such loads for a wave's keys
  static constexpr int kRowLoads = kQueryRows / kPerLoad / kWaves;   // and for its part of the staged query rows
  static constexpr int kBlockBytes = kQueryRows * kRowBytes;
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
  float per_group;   // 1 / group
  int slots;         // workgroups that run at a time
  int block;         // query rows of a block
  float scale_log2;  // scale log2 e
  float decay;
  float* partial;  // [parts of cut tiles][KV head][kTile]
  int32_t* status;
};

// ---------------------------------------------------------------------------------------------
// The layout of the work, derived by every workgroup from the lengths.
// ---------------------------------------------------------------------------------------------
// Tables in shared memory, of as many rows as there are.
struct Layout {
  int *first;  // parts of the rows before, of one KV head
  int *cut;    // those of them that are one of several of a tile
  int *start, *len, *keys;
  int rows, cap;  // cap: blocks of a part, at most
};
constexpr int layout_bytes(int rows) { return 4 * (5 * rows + 2); }

// Parts of each tile of a row.
__device__ __forceinline__ int row_parts(const MassArgs& a, int len, int cap) {
  return max(ceil_div(ceil_div(len * a.group, a.block), cap), 1);
}

__device__ __forceinline__ Layout make_layout(const MassArgs& a, int* memory, bool report) {
  __shared__ int scratch[4];
  __shared__ unsigned long long work;
  Layout y{memory, memory + a.rows + 1, memory + 2 * a.rows + 2, memory + 3 * a.rows + 2, memory + 4 * a.rows + 2, a.rows, 0};
  if (threadIdx.x == 0) work = 0;
  __syncthreads();
  unsigned long long mine = 0;
  for (int b = threadIdx.x; b < a.rows; b += kThreads) {
    int start = a.q_start[b], len = a.q_len[b], keys = a.t_len[b];
    uint32_t bits = keys > a.capacity ? kStatusLength : 0;
    if (len <= 0) {
      len = 0;
    } else if (start < 0 || len > a.tokens || start > a.tokens - len) {
      len = 0;
      bits |= kStatusRow;
    }
    if (bits && report && a.status) {
      __hip_atomic_fetch_or(a.status, static_cast<int>(bits), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    keys = len ? min(max(keys, 0), a.capacity) : 0;
    y.start[b] = start, y.len[b] = len, y.keys[b] = keys;
    mine += static_cast<unsigned long long>(ceil_div(keys, kTile)) * ceil_div(len * a.group, a.block);
  }
  if (mine) atomicAdd(&work, mine);
  __syncthreads();
  // A part has at least the share of the work at which kPartsPerSlot would fill every workgroup (which bounds the
  // partial sums).  Among the sizes that cut the longest rows evenly the one that ends first is taken: as
  // many rounds as all parts take, of a part's blocks and about two for what it costs beside them.  Of many rows it is the
  // least one.
  const unsigned long long most = static_cast<unsigned long long>(kPartsPerSlot) * a.slots;
  const unsigned long long share = (work * a.hkv + most - 1) / most;
  const int least = static_cast<int>(min(max(share, static_cast<unsigned long long>(kMinPart / a.block)), 1ull << 25));
  __shared__ int longest, cap;
  if (threadIdx.x == 0) longest = 0, cap = least;
  __syncthreads();
  int len = 0;
  for (int b = threadIdx.x; b < a.rows; b += kThreads) len = max(len, y.len[b]);
  len = ceil_div(len * a.group, a.block);
  if (len > least) atomicMax(&longest, len);
  __syncthreads();
  if (longest > least && a.rows <= kComparedRows && threadIdx.x < 64) {
    const int mine = max(ceil_div(longest, static_cast<int>(threadIdx.x) + 1), least);
    const float per_part = 1.f / static_cast<float>(mine);
    float parts = 0.f;
    for (int b = 0; b < a.rows; ++b) {
      const float blocks = static_cast<float>(ceil_div(y.len[b] * a.group, a.block));
      parts += static_cast<float>(ceil_div(y.keys[b], kTile)) * fmaxf(ceilf(blocks * per_part - 1e-3f), 1.f);
    }
    const float cost = ceilf(parts * static_cast<float>(a.hkv) / static_cast<float>(a.slots)) * static_cast<float>(mine + 2);
    const uint32_t best = wave_pick<false>(__float_as_uint(cost));
    const int lane = __builtin_ctzll(__ballot(__float_as_uint(cost) == best));
    if (static_cast<int>(threadIdx.x) == lane) cap = mine;
  }
  __syncthreads();
  y.cap = uniform(cap);
  build_row_prefix(a.rows, y.first, scratch, [&](int b) { return ceil_div(y.keys[b], kTile) * row_parts(a, y.len[b], y.cap); });
  build_row_prefix(a.rows, y.cut, scratch, [&](int b) {
    const int parts = row_parts(a, y.len[b], y.cap);
    return parts > 1 ? ceil_div(y.keys[b], kTile) * parts : 0;
  });
  return y;
}

// One part: a tile of a row's keys for one KV head, and which of its query rows.
struct Part {
  int head, row, start, len, keys, seen;
  int tile, part, parts, slot;
  int begin, end;  // blocks of query rows
};

// Query rows that see key t: [from, to) (rows hold at most 2^29 keys, and windows count as no more).
__device__ __forceinline__ int first_row(const MassArgs& a, const Part& p, int t) {
  return min(max(t - p.seen, 0), p.len) * a.group;
}
__device__ __forceinline__ int end_row(const MassArgs& a, const Part& p, int t) {
  return min(max(t - p.seen + a.window, 0), p.len) * a.group;
}

__device__ __forceinline__ Part part_at(const MassArgs& a, const Layout& y, int entry, int head) {
  Part p;
  p.head = head;
  p.row = uniform(find_row(y.first, y.rows, entry));
  p.start = uniform(y.start[p.row]), p.len = uniform(y.len[p.row]), p.keys = uniform(y.keys[p.row]);
  p.seen = p.keys - p.len;
  p.parts = row_parts(a, p.len, y.cap);
  const int in_row = entry - uniform(y.first[p.row]);
  p.tile = in_row / p.parts;
  p.part = in_row - p.tile * p.parts;
  p.slot = uniform(y.cut[p.row]) + in_row;
  // The blocks of query rows that see some key of the tile, and the part's share of them; one block where there
  // is none, of which no row counts.
  const int last_key = min((p.tile + 1) * kTile, p.keys) - 1;
  const int lo = first_row(a, p, p.tile * kTile) / a.block, hi = ceil_div(end_row(a, p, last_key), a.block);
  const int n = max(hi - lo, 0);
  p.begin = lo + static_cast<int>(static_cast<int64_t>(n) * p.part / p.parts);
  p.end = lo + static_cast<int>(static_cast<int64_t>(n) * (p.part + 1) / p.parts);
  return p;
}

// A part's blocks of query rows on their way to shared memory: the next block's first token in the query and
// the LSE, and its first row's head in the group.
struct Rows {
  uint64_t q, lse;
  int head, block, end;
};

template <int DT, int D, int R, bool WHOLE>
__global__ __launch_bounds__(kThreads, mass_groups(D, R)) void attention_mass_kernel(MassArgs args) {
  using M = Mass<D, R>;
  constexpr int kQueryRows = R, kHalves = R / 32;
  __shared__ __attribute__((aligned(512))) char lds[kTile * M::kRowBytes + 2 * M::kBlockBytes];
  __shared__ __attribute__((aligned(16))) float lse[2][kQueryRows];
  extern __shared__ int memory[];
  const Layout layout = make_layout(args, memory, blockIdx.x == 0);
  const int wave = uniform(threadIdx.x >> 6);
  const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const lds_char*)lds));
  const uint32_t keys_at = lds_at + wave * 32 * M::kRowBytes;
  const uint32_t rows_at = lds_at + kTile * M::kRowBytes + wave * M::kRowLoads * M::kPerLoad * M::kRowBytes;
  const int total = uniform(layout.first[args.rows]) * args.hkv;
  const float scale_log2 = args.scale_log2;

  // Lane i looks up the page of the wave's load i: kPerLoad neighbouring keys, which lie in one page where its
  // size is a multiple of kPerLoad (WHOLE).
  int page = 0, in = 0;
  // Parts go to the workgroups in turn, every other round backwards: their sizes fall or rise along the list.
  const int groups = gridDim.x;
  auto place_of = [&](int round) {
    return round * groups + (round & 1 ? groups - 1 - static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x));
  };
  auto find_part = [&](int i) {
    const MassArgs a = arguments<MassArgs>();
    const Part p = part_at(a, layout, i / a.hkv, i % a.hkv);
    const int load = WHOLE ? (fresh_thread() & 63) % M::kKeyLoads : 0;
    const int t = min(p.tile * kTile + wave * 32 + load * M::kPerLoad, (p.keys - 1) & ~(M::kPerLoad - 1));
    const int index = t / a.block_size;
    in = t - index * a.block_size;
    page = a.table[p.row * a.bt_stride + index];
    return p;
  };
  // Sends the wave's keys to its part of shared memory; returns the loads of a page out of range.
  auto send_keys = [&](const Part& p) {
    const MassArgs a = arguments<MassArgs>();
    const int lane = fresh_thread() & 63, piece = lane % M::kPieces, mine = lane / M::kPieces;
    const uint32_t token_bytes = a.k_token;
    const uint64_t cache = reinterpret_cast<uint64_t>(a.k) + p.head * a.k_head;
    uint32_t bad = 0;
    if constexpr (WHOLE) {
      const bool exists = static_cast<unsigned>(page) < static_cast<unsigned>(a.num_blocks);
      bad = static_cast<uint32_t>(__ballot(!exists)) & static_cast<uint32_t>((1ull << M::kKeyLoads) - 1);
      const uint64_t place = cache + static_cast<uint32_t>(exists ? page : 0) * a.k_block + static_cast<uint32_t>(in) * token_bytes;
#pragma unroll
      for (int i = 0; i < M::kKeyLoads; ++i) {
        load_lds<0>(lane_value(place, i), mine * token_bytes + 16 * (piece ^ key_turn<D>(i * M::kPerLoad + mine)),
                    keys_at + i * M::kPerLoad * M::kRowBytes);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < M::kKeyLoads; ++i) {
        const int key = i * M::kPerLoad + mine, t = min(p.tile * kTile + wave * 32 + key, p.keys - 1);
        const int index = t / a.block_size, found = a.table[p.row * a.bt_stride + index];
        const bool exists = static_cast<unsigned>(found) < static_cast<unsigned>(a.num_blocks);
        const uint64_t from = cache + static_cast<uint32_t>(exists ? found : 0) * a.k_block +
                              static_cast<uint32_t>(t - index * a.block_size) * token_bytes;
        for (int j = 0; j < M::kPerLoad; ++j) {  // a bit a key
          bad |= (__ballot(!exists) >> (j * M::kPieces)) & 1 ? 1u << (i * M::kPerLoad + j) : 0u;
        }
        load_lds<0>(from + 16 * (piece ^ key_turn<D>(key)), uniform(keys_at + i * M::kPerLoad * M::kRowBytes));
      }
    }
    if (bad && a.status) {
      __hip_atomic_fetch_or(a.status, static_cast<int>(kStatusPage), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    return bad;
  };

  // Where the lane's pieces of a block lie after the block's first token, and its row's LSE, in bytes.  They
  // depend on the first row's head alone, and on where the last row lies in the last block.
  uint32_t row_offset[M::kRowLoads], lse_offset = 0;
  int placed = -1;
  auto place_rows = [&](int head, int last) {
    const MassArgs a = arguments<MassArgs>();
    const int lane = fresh_thread() & 63, piece = lane % M::kPieces;
    // (n + 0.5) / group in floating point gives the exact quotient for n < 2^22.
    auto split = [&](int row, int& in_group) {
      const int n = head + min(row, last), t = static_cast<int>((static_cast<float>(n) + 0.5f) * a.per_group);
      in_group = n - t * a.group;
      return t;
    };
    int in_group;
#pragma unroll
    for (int i = 0; i < M::kRowLoads; ++i) {
      const int row = (wave * M::kRowLoads + i) * M::kPerLoad + lane / M::kPieces, t = split(row, in_group);
      row_offset[i] = 2 * (t * static_cast<uint32_t>(a.q_row) + in_group * static_cast<uint32_t>(a.q_head)) +
                      16 * (piece ^ key_turn<D>(row));
    }
    const int t = split(lane & (kQueryRows - 1), in_group);
    lse_offset = 4 * (t * static_cast<uint32_t>(a.l_row) + in_group * static_cast<uint32_t>(a.l_head));
    placed = last < kQueryRows - 1 ? -1 : head;
  };
  const int block_heads = kQueryRows % args.group;
  const int64_t block_q = 2 * (kQueryRows / args.group) * args.q_row, block_lse = 4 * (kQueryRows / args.group) * args.l_row;
  auto start_rows = [&](const Part& p) {
    const MassArgs a = arguments<MassArgs>();
    Rows r;
    // One block where there is none, of which no row counts.
    r.block = min(p.begin, ceil_div(p.len * a.group, kQueryRows) - 1);
    r.end = max(p.end, r.block + 1);
    const int token = r.block * kQueryRows / a.group;
    r.head = r.block * kQueryRows - token * a.group;
    r.q = reinterpret_cast<uint64_t>(a.q + (p.start + token) * a.q_row + p.head * a.group * a.q_head);
    r.lse = reinterpret_cast<uint64_t>(a.lse + (p.start + token) * a.l_row + p.head * a.group * a.l_head);
    return r;
  };
  float next_lse = 0.f;  // lane of wave 0: of a row of the block on its way
  // Sends a block of query rows to a half of their shared memory; rows past the last one (`last`) repeat it.
  auto send_rows = [&](Rows& r, int last, int half) {
    if (placed != r.head || last < kQueryRows - 1) place_rows(r.head, last);
#pragma unroll
    for (int i = 0; i < M::kRowLoads; ++i) {
      if ((wave * M::kRowLoads + i) * M::kPerLoad > last) break;
      load_lds<0>(r.q, row_offset[i], uniform(rows_at + half * M::kBlockBytes + i * M::kPerLoad * M::kRowBytes));
    }
    typedef const __attribute__((address_space(1))) float* global_float;
    if (wave == 0) next_lse = *(global_float)(r.lse + lse_offset);
    r.q += block_q, r.lse += block_lse, r.head += block_heads;
    ++r.block;
    if (block_heads) {
      const MassArgs a = arguments<MassArgs>();
      if (r.head >= a.group) {
        r.head -= a.group;
        r.q += 2 * a.q_row, r.lse += 4 * a.l_row;
      }
    }
  };

  int round = 0, i = place_of(0);
  if (i >= total) return;
  // While a part is computed the keys and first query rows of the next one are on their way, and the pages of the
  // one after it are looked up.
  Part u = find_part(i), v = u;
  uint32_t bad = send_keys(u), bad_ahead = 0;
  Rows rows = start_rows(u);
  int block = rows.block, last_row = u.len * args.group - 1;
  send_rows(rows, last_row - block * kQueryRows, 0);
  i = place_of(++round);
  if (i < total) v = find_part(i);
  int half = 0;
  for (;;) {
    const int lane = threadIdx.x & 63, end_of_rows = last_row + 1;
    int from, to, all_from, all_to;  // rows that see the lane's key, and that see all of the wave's
    {
      const MassArgs a = arguments<MassArgs>();
      const int t0 = u.tile * kTile + wave * 32, t = t0 + (lane & 31);
      const int part_from = u.begin * kQueryRows, part_to = u.end * kQueryRows;
      from = max(first_row(a, u, t), part_from), to = t < u.keys ? min(end_row(a, u, t), part_to) : 0;
      all_from = max(first_row(a, u, t0 + 31), part_from);
      all_to = t0 + 31 < u.keys ? min(end_row(a, u, t0), part_to) : 0;
    }
    u32x4 k[M::kSteps];
    float sum = 0.f;
    const int begin = block, end = rows.end;
    for (; block < end; ++block) {
      wait_loads();
      if (wave == 0 && lane < kQueryRows) {
        // A query head that saw nothing adds nothing.
        lse[half][lane] = next_lse == -INFINITY ? INFINITY : next_lse * kLog2eP;
      }
      lds_barrier();
      if (block == begin) {
        const int key = lane & 31;
        const char* at = lds + (wave * 32 + key) * M::kRowBytes;
#pragma unroll
        for (int s = 0; s < M::kSteps; ++s) {
          k[s] = *reinterpret_cast<const u32x4*>(at + 16 * ((2 * s + (lane >> 5)) ^ key_turn<D>(key)));
        }
        if (bad) {
          const bool mine = (bad >> (WHOLE ? key / M::kPerLoad : key)) & 1;
#pragma unroll
          for (int s = 0; s < M::kSteps; ++s) k[s] = mine ? u32x4{0, 0, 0, 0} : k[s];
        }
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // the next keys may come
      }
      if (block + 1 < end) {
        send_rows(rows, last_row - (block + 1) * kQueryRows, half ^ 1);
      } else if (i < total) {
        bad_ahead = send_keys(v);
        rows = start_rows(v);
        last_row = v.len * arguments<MassArgs>().group - 1;
        send_rows(rows, last_row - rows.block * kQueryRows, half ^ 1);
      }
      // Scores of the query rows with the wave's keys, 32 rows at a time: the products of the second run while the
      // first are weighed.
      const int thread = fresh_thread() & 63, row = thread & 31, upper = thread >> 5;
      const char* staged = lds + kTile * M::kRowBytes + half * M::kBlockBytes;
      const uint32_t at = row * M::kRowBytes + 16 * (upper ^ key_turn<D>(row));
      const int r0 = block * kQueryRows;
      auto score = [&](int b, f32x16& sc) {
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = 0.f;
#pragma unroll
        for (int s = 0; s < M::kSteps; ++s) {
          sc = mfma32<DT>(*reinterpret_cast<const u32x4*>(staged + (at ^ (32 * s)) + 32 * b * M::kRowBytes), k[s], sc);
        }
      };
      auto weigh = [&](int b, const f32x16& sc, bool masked) {
        float w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float x = lse[half][32 * b + 8 * (e >> 2) + 4 * upper + (e & 3)];
          w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], scale_log2, -x));
        }
        if (masked) {
          const int first = from - r0 - 32 * b - 4 * upper;
          const unsigned count = max(to - from, 0);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if (static_cast<unsigned>(8 * (e >> 2) + (e & 3) - first) >= count) w[e] = 0.f;
          }
        }
#pragma unroll
        for (int n = 8; n >= 1; n >>= 1) {
#pragma unroll
          for (int e = 0; e < n; ++e) w[e] += w[e + n];
        }
        sum += w[0];
      };
      if (kHalves == 2 && r0 >= all_from && r0 + kQueryRows <= all_to) {
        // The rows are read ahead of the first products, those of the second between them, and the first are weighed
        // between the second products.  (The compiler orders this otherwise, left to itself.)
        u32x4 rows0[M::kSteps], rows1[M::kSteps];
        f32x4 lse0[4], lse1[4];
        auto read = [&](int b, int s) { return *reinterpret_cast<const u32x4*>(staged + (at ^ (32 * s)) + 32 * b * M::kRowBytes); };
        auto read_lse = [&](int b, int e) { return *reinterpret_cast<const f32x4*>(&lse[half][32 * b + 8 * e + 4 * upper]); };
        f32x16 sc0, sc1;
#pragma unroll
        for (int e = 0; e < 16; ++e) sc0[e] = sc1[e] = 0.f;
#pragma unroll
        for (int s = 0; s < M::kSteps; ++s) rows0[s] = read(0, s);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < M::kSteps; ++s) {
          sc0 = mfma32<DT>(rows0[s], k[s], sc0);
          rows1[s] = read(1, s);
          if (s < 4) lse0[s] = read_lse(0, s);
          __builtin_amdgcn_sched_barrier(0);
        }
        constexpr int kEach = 16 / M::kSteps;
        float w0 = 0.f, w1 = 0.f;
        auto weigh = [&](const f32x16& sc, const f32x4(&x)[4], int e) {
          return __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], scale_log2, -x[e >> 2][e & 3]));
        };
#pragma unroll
        for (int s = 0; s < M::kSteps; ++s) {
          sc1 = mfma32<DT>(rows1[s], k[s], sc1);
          if (s < 4) lse1[s] = read_lse(1, s);
#pragma unroll
          for (int e = 0; e < kEach; ++e) {
            const float x = weigh(sc0, lse0, s * kEach + e);
            if (e & 1) w1 += x; else w0 += x;
          }
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int e = 0; e < 16; e += 2) w0 += weigh(sc1, lse1, e), w1 += weigh(sc1, lse1, e + 1);
        sum += w0 + w1;
      } else {
#pragma unroll
        for (int b = 0; b < kHalves; ++b) {
          if (r0 + 32 * b >= end_of_rows) break;
          f32x16 sc;
          score(b, sc);
          weigh(b, sc, r0 < all_from || r0 + kQueryRows > all_to);
        }
      }
      half ^= 1;
    }
    sum += other_half(sum);
    {
      const MassArgs a = arguments<MassArgs>();
      const int in_tile = wave * 32 + lane, t = u.tile * kTile + in_tile;
      if (lane < 32 && t < u.keys) {
        if (u.parts > 1) {
          a.partial[(static_cast<int64_t>(u.slot) * a.hkv + u.head) * kTile + in_tile] = sum;
        } else {
          const float old = a.previous ? a.decay * a.previous[u.row * a.p_row + u.head * a.p_head + t] : 0.f;
          a.mass[u.row * a.m_row + u.head * a.m_head + t] = old + sum;
        }
      }
    }
    if (i >= total) break;
    u = v;
    bad = bad_ahead;
    block = rows.block - 1;
    i = place_of(++round);
    if (i < total) v = find_part(i);
  }
}

// Adds up the parts of cut tiles, a thread a key.
__global__ __launch_bounds__(kThreads) void mass_join_kernel(MassArgs a) {
  extern __shared__ int memory[];
  const Layout layout = make_layout(a, memory, false);
  const int total = uniform(layout.cut[a.rows]) * a.hkv;
  for (int i = blockIdx.x; i < total; i += gridDim.x) {
    const int entry = i / a.hkv, head = i - entry * a.hkv;
    // The rows without cut tiles have no entries here.
    const int row = uniform(find_row(layout.cut, a.rows, entry));
    const Part p = part_at(a, layout, uniform(layout.first[row]) + entry - uniform(layout.cut[row]), head);
    const int t = p.tile * kTile + threadIdx.x;
    if (p.part || threadIdx.x >= kTile || t >= p.keys) continue;
    float sum = a.previous ? a.decay * a.previous[p.row * a.p_row + head * a.p_head + t] : 0.f;
    for (int j = 0; j < p.parts; ++j) sum += a.partial[(static_cast<int64_t>(p.slot + j) * a.hkv + head) * kTile + threadIdx.x];
    a.mass[p.row * a.m_row + head * a.m_head + t] = sum;
  }
}

// Parts of cut tiles: a row's tiles have at most twice the parts that their blocks fill, so at most 2
// kPartsPerSlot for each workgroup that runs at a time, all KV heads together.
int64_t partial_parts() { return 2LL * kPartsPerSlot * kMostGroups * device_cu_count() + 1; }
size_t mass_workspace_bytes() { return static_cast<size_t>(partial_parts()) * kTile * sizeof(float); }

template <int DT, int D, int R>
void launch_block(hipStream_t stream, const MassArgs& a) {
  if (a.block_size % Mass<D, R>::kPerLoad == 0) {
    attention_mass_kernel<DT, D, R, true><<<a.slots, kThreads, layout_bytes(a.rows), stream>>>(a);
  } else {
    attention_mass_kernel<DT, D, R, false><<<a.slots, kThreads, layout_bytes(a.rows), stream>>>(a);
  }
}

template <int DT, int D>
void launch(hipStream_t stream, const MassArgs& a) {
  if (a.block == 32) launch_block<DT, D, 32>(stream, a);
  else launch_block<DT, D, 64>(stream, a);
}

template <int DT>
void launch_dim(hipStream_t stream, int d, const MassArgs& a) {
  if (d == 64) launch<DT, 64>(stream, a);
  else if (d == 128) launch<DT, 128>(stream, a);
  else launch<DT, 256>(stream, a);
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
  DS_SUPPORTED(capacity <= (1 << 29), "rows of at most 2^29 keys");
  DS_SUPPORTED(d->tokens <= (1 << 20), "at most 2^20 query tokens");
  DS_SUPPORTED(group <= (1 << 16), "at most 2^16 query heads for a KV head");
  // Places within a block of query rows are 32-bit byte counts, the heads of one more token included.
  const auto spans = [&](int64_t row, int64_t head) {
    return std::max<int64_t>(row, -row) * (kMostRows / group + 2) + std::max<int64_t>(head, -head) * group < (1 << 30);
  };
  DS_SUPPORTED(spans(d->q_row_stride, d->q_head_stride) && d->lse_token_stride >= 0 && d->lse_head_stride >= 0 &&
                   spans(d->lse_token_stride, d->lse_head_stride),
               "query and LSE strides of at most 2^30 elements a block of rows");
  // Parts are counted in 32 bits.
  const int64_t tiles = static_cast<int64_t>(d->rows) * ((capacity + kTile - 1) / kTile);
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
  a.per_group = 1.f / static_cast<float>(group);
  a.block = static_cast<int64_t>(d->tokens) * group <= 32LL * d->rows ? 32 : 64;
  a.slots = mass_groups(d->head_dim, a.block) * device_cu_count();
  a.scale_log2 = d->scale * kLog2eP;
  a.decay = d->decay;
  a.partial = static_cast<float*>(d->workspace);
  a.status = d->status;
  if (d->dtype == DS_BF16) launch_dim<DS_BF16>(stream, d->head_dim, a);
  else launch_dim<DS_FP16>(stream, d->head_dim, a);
  // Fewer query rows than a part's make no parts.
  if (static_cast<int64_t>(d->tokens) * group > kMinPart) {
    mass_join_kernel<<<a.slots, kThreads, layout_bytes(a.rows), stream>>>(a);
  }
  return check_launch("ds_attention_mass");
}

}  // namespace
}  // namespace ds355

extern "C" size_t ds_attention_mass_workspace_bytes(void) { return ds355::mass_workspace_bytes(); }

extern "C" int ds_attention_mass(ds_stream_t stream, const ds_attention_mass_desc* desc) {
  return ds355::attention_mass_impl(reinterpret_cast<hipStream_t>(stream), desc);
}

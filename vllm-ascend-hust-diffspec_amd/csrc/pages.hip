// Pages of a paged cache: copying, forking rows that share them, growing and freeing rows, compacting.
//
// The reference takes its pages and block tables from the serving engine's host allocator
// (diffspec/runtime.py:869-875 keeps the table it is handed).  Here the state lives on the device, so a
// step can fork, cut back and grow rows without a host round trip:
//   ref_counts [num_pages]         rows that hold the page; 0 = free
//   block_table [rows, width]      a row's pages in order, -1 behind its last
// Free pages are always taken in ascending order, for the call's rows in their order, so a call's result
// depends on the state alone.
//
// The bookkeeping is latency-bound (a few thousand words); the copies are bound by memory.  One
// workgroup takes pages (ranks need one order), every workgroup releases, shares or copies.  A fork's
// last workgroup to have released takes the pages, which saves a launch.  Measured: a fork of 4 rows
// 6.3 + 3.6 us (checks and pages, then entries and copies), of 248 rows of up to 4000 tokens, a page of each
// copied in 8 caches of 32 KiB, 9.0 + 12.8 to 14.4, both with children that share the parent's entries already
// (248 rows with 153 pages copied: the same fork again 19.3 us, with another parent for each row every time
// 24.0); 128 rows cut back and grown again 3.5 + 9.6; copies 4.9 TB/s both ways (a large plain copy reaches 5.1); a
// compaction's plan over 4096 pages 7.0 and its moves 5.3 TB/s.
#include "ds355_common.h"

namespace ds355 {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreadsP = 1024;
constexpr int kMaxList = 4096;   // rows of a table, and entries of a call's lists
constexpr int kMaxPages = INT_MAX - (1 << 14);  // the scans look up to 12288 pages ahead in 32 bits
constexpr int kCopyThreads = 256;
constexpr int kPiece = 4096;     // bytes that a wave copies at a time
constexpr int32_t kBadRow = 1;     // a row (or a list entry) the call leaves out
constexpr int32_t kNoPages = 2;    // the pool ran out of free pages
constexpr int32_t kBadPage = 4;    // a page id is outside the pool, or its count was 0 when it was freed

// Workspace words: a counter (0 between launches), results of a compaction, then a word or two per
// list entry or page.
enum { kHdrDone = 0, kHdrMoves = 1, kHdrLive = 2, kHeaderWords = 64 };

struct Table {
  int32_t* entries;
  int64_t stride;
  int rows, width;
};

struct Caches {
  const int64_t* list;  // per cache: address, bytes between pages, bytes of a page, 1 if all whole 16-byte vectors
  int count;
  int pieces;  // pieces of the largest page
};

__device__ __forceinline__ void raise(int32_t* status, int32_t bits) {
  if (status && bits) __hip_atomic_fetch_or(status, bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ int ceil_div(int a, int b) { return a / b + (a % b != 0); }

// One row less holds the page; the status bits of a page that no row can hold.
__device__ __forceinline__ int32_t drop(int page, int32_t* refs, int num_pages) {
  if (page >= num_pages) return kBadPage;
  if (atomicSub(refs + page, 1) > 0) return 0;
  atomicAdd(refs + page, 1);
  return kBadPage;
}

__device__ __forceinline__ bool block_any(bool v) { return __syncthreads_or(v) != 0; }

// Exclusive scan over the workgroup; `total` is the sum.
__device__ __forceinline__ int scan1024(int v, int* scratch, int& total) {
  const int inc = wave_inclusive_scan(v), wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 63) scratch[wave] = inc;
  __syncthreads();
  int base = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreadsP / 64; ++w) {
    const int s = scratch[w];
    if (w < wave) base += s;
    total += s;
  }
  return base + inc - v;
}

// Four counts from page `at` on (read at device scope where other workgroups of this launch change
// them); pages past the pool count as held.
template <bool COHERENT>
__device__ __forceinline__ u32x4 counts_at(const int32_t* refs, int at, int num_pages) {
  u32x4 v = {1, 1, 1, 1};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (at + i < num_pages) v[i] = static_cast<uint32_t>(COHERENT ? coherent_load(refs + at + i) : refs[at + i]);
  }
  return v;
}

// Calls take(rank, page) for the first `need` free pages in ascending order; returns how many there were.
template <bool COHERENT, typename Take>
__device__ __forceinline__ int take_pages(int32_t* refs, int num_pages, int need, int* scratch, Take take) {
  int found = 0;
  u32x4 next = counts_at<COHERENT>(refs, 4 * threadIdx.x, num_pages);
  for (int base = 0; base < num_pages && found < need; base += 4 * kThreadsP) {
    const u32x4 v = next;
    const int at = base + 4 * static_cast<int>(threadIdx.x);
    next = counts_at<COHERENT>(refs, at + 4 * kThreadsP, num_pages);
    int mine = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) mine += v[i] == 0;
    int total;
    int rank = found + scan1024(mine, scratch, total);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (v[i] == 0) {
        if (rank < need) take(rank, at + i);
        ++rank;
      }
    }
    found += total;
  }
  return min(found, need);
}

// ---------------------------------------------------------------------------------------------
// Copies: a wave moves one piece (pair, cache, 4 KiB) at a time.
// ---------------------------------------------------------------------------------------------
// Cached loads and non-temporal stores, 64 workgroups a CU: us for 200 pages of 12 x 32 KiB caches (157 MB
// both ways) / a compaction that moves 1.0 GB: 31.9 / 200; with cached stores and 16 a CU 38.4 / 219,
// non-temporal stores and 16 a CU 32.4 / 210, non-temporal loads too 33.4 / 205.
__device__ __forceinline__ void copy_piece(const Caches& c, int cache, int piece, int64_t src, int64_t dst) {
  const int64_t* d = c.list + 4 * cache;
  const int64_t bytes = d[2], from = static_cast<int64_t>(piece) * kPiece;
  const int n = static_cast<int>(min(static_cast<int64_t>(kPiece), bytes - from));
  if (n <= 0) return;
  const char* s = reinterpret_cast<const char*>(d[0]) + src * d[1] + from;
  char* t = reinterpret_cast<char*>(d[0]) + dst * d[1] + from;
  const int lane = threadIdx.x & 63;
  if (d[3]) {
    u32x4 v[kPiece / 1024];
#pragma unroll
    for (int i = 0; i < kPiece / 1024; ++i) {
      if (16 * (lane + 64 * i) < n) v[i] = *reinterpret_cast<const u32x4*>(s + 16 * (lane + 64 * i));
    }
#pragma unroll
    for (int i = 0; i < kPiece / 1024; ++i) {
      u32x4* to = reinterpret_cast<u32x4*>(t + 16 * (lane + 64 * i));
      if (16 * (lane + 64 * i) < n) __builtin_nontemporal_store(v[i], to);
    }
  } else {
    for (int i = lane; i < n; i += 64) t[i] = s[i];
  }
}

// Work items (pair, cache, piece) in that order, dealt to the waves of the workgroups from `first` on.
template <typename Pair>
__device__ __forceinline__ void copy_all(const Caches& c, int64_t pairs, int first, Pair pair) {
  const int64_t per_pair = static_cast<int64_t>(c.count) * c.pieces;
  const int waves = static_cast<int>(blockDim.x >> 6);
  const int64_t step = static_cast<int64_t>(gridDim.x - first) * waves;
  for (int64_t w = static_cast<int64_t>(blockIdx.x - first) * waves + (threadIdx.x >> 6); w < pairs * per_pair; w += step) {
    const int64_t i = w / per_pair;
    const int rest = static_cast<int>(w - i * per_pair);
    int64_t src, dst;
    if (pair(i, src, dst)) copy_piece(c, rest / c.pieces, rest % c.pieces, src, dst);
  }
}

__global__ __launch_bounds__(kCopyThreads) void copy_pages_kernel(Caches c, const int32_t* src, const int32_t* dst,
                                                                  int count, int num_pages, int32_t* status) {
  copy_all(c, count, 0, [&](int64_t i, int64_t& s, int64_t& d) {
    s = src[i], d = dst[i];
    if (s < 0 || s >= num_pages || d < 0 || d >= num_pages) {
      raise(status, kBadPage);
      return false;
    }
    return s != d;
  });
}

// ---------------------------------------------------------------------------------------------
// Fork
// ---------------------------------------------------------------------------------------------
struct ForkArgs {
  Caches caches;
  Table table;
  int32_t* refs;
  int num_pages;
  const int32_t* parents;
  const int32_t* children;
  const int32_t* lens;
  int count, block_size;
  int32_t* header;
  int32_t* page;  // per pair: its new page, or one of the words below
  int32_t* status;
};
constexpr int kNoPage = -1, kLeftOut = -2, kNoneFree = -3;

// One workgroup per pair: checks it, gives the child's pages back; the last one takes the new pages.
__global__ __launch_bounds__(kThreadsP) void fork_release_kernel(ForkArgs a) {
  __shared__ int scratch[kThreadsP / 64];
  __shared__ int order[kMaxList];
  const int i = blockIdx.x;
  const int parent = a.parents[i], child = a.children[i], len = a.lens[i];
  bool bad = parent < 0 || parent >= a.table.rows || child < 0 || child >= a.table.rows || parent == child || len < 0;
  int pages = 0;
  if (!bad) {
    pages = ceil_div(len, a.block_size);
    bad = pages > a.table.width;
  }
  for (int j = threadIdx.x; j < a.count; j += kThreadsP) {
    bad |= (j < i && a.children[j] == child) || a.parents[j] == child;
  }
  bad = block_any(bad);
  if (!bad) {
    const int32_t* e = a.table.entries + static_cast<int64_t>(parent) * a.table.stride;
    for (int c = threadIdx.x; c < pages; c += kThreadsP) bad |= e[c] < 0 || e[c] >= a.num_pages;
    bad = block_any(bad);
  }
  if (!bad) {
    // Entries that the child has already (forked from this parent before) stay, with their counts: the
    // parent holds those pages, so whether they are given back and shared again makes no difference.
    const int full = len / a.block_size;
    int32_t* e = a.table.entries + static_cast<int64_t>(child) * a.table.stride;
    const int32_t* from = a.table.entries + static_cast<int64_t>(parent) * a.table.stride;
    int32_t bits = 0;
    for (int c = threadIdx.x; c < a.table.width; c += kThreadsP) {
      const int page = e[c];
      if (page < 0 || (c < full && page == from[c])) continue;
      e[c] = -1;
      bits |= drop(page, a.refs, a.num_pages);
    }
    raise(a.status, bits);
  }
  if (threadIdx.x == 0) {
    if (bad) raise(a.status, kBadRow);
    coherent_store(a.page + i, bad ? kLeftOut : len % a.block_size ? 0 : kNoPage);
  }
  // What the last workgroup reads of the others (counts, page words) is written past the caches, so it has
  // arrived once the writes are acknowledged.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  __shared__ int done;
  if (threadIdx.x == 0) done = __hip_atomic_fetch_add(a.header + kHdrDone, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (done != a.count - 1) return;
  int need = 0;
  for (int base = 0; base < a.count; base += kThreadsP) {
    const int j = base + static_cast<int>(threadIdx.x);
    const bool wants = j < a.count && coherent_load(a.page + j) == 0;
    int total;
    const int rank = need + scan1024(wants, scratch, total);
    if (wants) order[rank] = j;
    need += total;
  }
  __syncthreads();
  const int found = take_pages<true>(a.refs, a.num_pages, need, scratch, [&](int rank, int page) {
    a.page[order[rank]] = page;
    a.refs[page] = 1;
  });
  for (int r = found + static_cast<int>(threadIdx.x); r < need; r += kThreadsP) a.page[order[r]] = kNoneFree;
  if (threadIdx.x == 0) {
    if (found < need) raise(a.status, kNoPages);
    a.header[kHdrDone] = 0;
  }
}

// The first `count` workgroups write the children's rows, the others copy the partial pages.
__global__ __launch_bounds__(kCopyThreads) void fork_share_kernel(ForkArgs a) {
  if (static_cast<int>(blockIdx.x) < a.count) {
    const int i = blockIdx.x, page = a.page[i];
    if (page == kLeftOut) return;
    const int full = a.lens[i] / a.block_size;
    const int32_t* from = a.table.entries + static_cast<int64_t>(a.parents[i]) * a.table.stride;
    int32_t* to = a.table.entries + static_cast<int64_t>(a.children[i]) * a.table.stride;
    for (int c = threadIdx.x; c < full; c += kCopyThreads) {
      const int p = from[c], had = to[c];
      if (page == kNoneFree) {  // the child stays empty
        if (had >= 0) atomicSub(a.refs + had, 1);
        to[c] = -1;
      } else if (had != p) {
        to[c] = p;
        atomicAdd(a.refs + p, 1);
      }
    }
    if (threadIdx.x == 0 && page >= 0) to[full] = page;
    return;
  }
  copy_all(a.caches, a.count, a.count, [&](int64_t i, int64_t& s, int64_t& d) {
    d = a.page[i];
    if (d < 0) return false;
    s = a.table.entries[static_cast<int64_t>(a.parents[i]) * a.table.stride + a.lens[i] / a.block_size];
    return true;
  });
}

// ---------------------------------------------------------------------------------------------
// Growing and freeing rows
// ---------------------------------------------------------------------------------------------
// One workgroup: rows' needs, then free pages to entries.
__global__ __launch_bounds__(kThreadsP) void extend_kernel(Table t, int32_t* refs, int num_pages, const int32_t* rows,
                                                           const int32_t* lens, int count, int block_size,
                                                           int32_t* status) {
  __shared__ int scratch[kThreadsP / 64];
  __shared__ int first[kMaxList];      // first list entry of each row
  __shared__ int before[kMaxList + 1]; // pages that the entries before need
  __shared__ int held[kMaxList];
  for (int r = threadIdx.x; r < t.rows; r += kThreadsP) first[r] = INT_MAX;
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += kThreadsP) {
    if (rows[i] >= 0 && rows[i] < t.rows) atomicMin(&first[rows[i]], i);
  }
  __syncthreads();
  int need = 0;
  for (int base = 0; base < count; base += kThreadsP) {
    const int i = base + static_cast<int>(threadIdx.x);
    int want = 0;
    if (i < count) {
      const int row = rows[i], len = lens[i];
      bool bad = row < 0 || row >= t.rows || first[row < 0 || row >= t.rows ? 0 : row] != i || len < 0;
      int pages = 0;
      if (!bad) {
        pages = ceil_div(len, block_size);
        bad = pages > t.width;
      }
      if (bad) {
        raise(status, kBadRow);
      } else {
        // The row's pages are its leading entries.  A thread halves for their end: 128 rows of 4097 tokens in
        // pages of 16 take 9.2 us, where waves that look at 64 places of several rows at once take 13.
        const int32_t* e = t.entries + static_cast<int64_t>(row) * t.stride;
        int lo = 0, hi = pages;
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (e[mid] >= 0) lo = mid + 1; else hi = mid;
        }
        held[i] = lo;
        want = pages - lo;
      }
    }
    int total;
    const int at = need + scan1024(want, scratch, total);
    if (i < count) before[i] = at;
    need += total;
  }
  if (threadIdx.x == 0) before[count] = need;
  __syncthreads();
  auto entry = [&](int rank) {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (before[mid] <= rank) lo = mid; else hi = mid - 1;
    }
    return lo;
  };
  const int found = take_pages<false>(refs, num_pages, need, scratch, [&](int rank, int page) {
    const int i = entry(rank);
    t.entries[static_cast<int64_t>(rows[i]) * t.stride + held[i] + rank - before[i]] = page;
    refs[page] = 1;
  });
  if (found == need) return;
  // Too few: the row that got a part gives it back (the rows after it got nothing).
  __syncthreads();
  const int i = entry(found);
  for (int r = before[i] + static_cast<int>(threadIdx.x); r < found; r += kThreadsP) {
    int32_t* e = t.entries + static_cast<int64_t>(rows[i]) * t.stride + held[i] + r - before[i];
    refs[*e] = 0;
    *e = -1;
  }
  if (threadIdx.x == 0) raise(status, kNoPages);
}

__global__ __launch_bounds__(256) void free_kernel(Table t, int32_t* refs, int num_pages, const int32_t* rows,
                                                   const int32_t* keep, int block_size, int32_t* status) {
  const int row = rows[blockIdx.x], len = keep ? keep[blockIdx.x] : 0;
  if (row < 0 || row >= t.rows || len < 0) {
    if (threadIdx.x == 0) raise(status, kBadRow);
    return;
  }
  // Each entry is taken out with one exchange, so that a row named twice gives its pages back once.
  int32_t* e = t.entries + static_cast<int64_t>(row) * t.stride;
  int32_t bits = 0;
  for (int c = ceil_div(len, block_size) + static_cast<int>(threadIdx.x); c < t.width; c += blockDim.x) {
    if (e[c] < 0) continue;
    const int page = atomicExch(e + c, -1);
    if (page >= 0) bits |= drop(page, refs, num_pages);
  }
  raise(status, bits);
}

// ---------------------------------------------------------------------------------------------
// Compaction: the k-th held page at or past the number of held pages moves to the k-th free page below it.
// ---------------------------------------------------------------------------------------------
struct CompactArgs {
  Caches caches;
  Table table;
  int32_t* refs;
  int num_pages;
  int32_t* page_map;  // new place of each page, -1 for free ones
  int32_t* header;
  int32_t* from;  // [num_pages] pages that move, in ascending order
  int32_t* to;    // [num_pages]
  int32_t* status;
};

__global__ __launch_bounds__(kThreadsP) void compact_plan_kernel(CompactArgs a) {
  __shared__ int scratch[kThreadsP / 64];
  int mine = 0, live;
  for (int at = 4 * threadIdx.x; at < a.num_pages; at += 4 * kThreadsP) {
    const u32x4 v = counts_at<false>(a.refs, at, a.num_pages);
#pragma unroll
    for (int i = 0; i < 4; ++i) mine += at + i < a.num_pages && v[i] != 0;
  }
  scan1024(mine, scratch, live);
  int holes = 0, moves = 0;
  for (int base = 0; base < a.num_pages; base += 4 * kThreadsP) {
    const int at = base + 4 * static_cast<int>(threadIdx.x);
    const u32x4 v = counts_at<false>(a.refs, at, a.num_pages);
    int h = 0, m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (at + i < a.num_pages) {
        h += at + i < live && v[i] == 0;
        m += at + i >= live && v[i] != 0;
        a.page_map[at + i] = v[i] != 0 ? at + i : -1;
      }
    }
    int total;
    int hr = holes + scan1024(h, scratch, total);
    holes += total;
    int mr = moves + scan1024(m, scratch, total);
    moves += total;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (at + i < a.num_pages) {
        if (at + i < live && v[i] == 0) a.to[hr++] = at + i;
        if (at + i >= live && v[i] != 0) a.from[mr++] = at + i;
      }
    }
  }
  __syncthreads();
  for (int k = threadIdx.x; k < moves; k += kThreadsP) {
    const int s = a.from[k], d = a.to[k];
    a.page_map[s] = d;
    a.refs[d] = a.refs[s];
    a.refs[s] = 0;
  }
  if (threadIdx.x == 0) {
    a.header[kHdrMoves] = moves;
    a.header[kHdrLive] = live;
  }
}

__global__ __launch_bounds__(kCopyThreads) void compact_move_kernel(CompactArgs a) {
  const int64_t cells = static_cast<int64_t>(a.table.rows) * a.table.width;
  const int live = a.header[kHdrLive];
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kCopyThreads + threadIdx.x; i < cells;
       i += static_cast<int64_t>(gridDim.x) * kCopyThreads) {
    const int64_t row = i / a.table.width;
    int32_t* e = a.table.entries + row * a.table.stride + (i - row * a.table.width);
    const int p = *e;
    if (p >= a.num_pages) raise(a.status, kBadPage);
    else if (p >= live) *e = a.page_map[p];
  }
  copy_all(a.caches, a.header[kHdrMoves], 0, [&](int64_t i, int64_t& s, int64_t& d) {
    s = a.from[i], d = a.to[i];
    return true;
  });
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
int copy_blocks(const Caches& c, int64_t pairs) {
  const int64_t pieces = pairs * c.count * c.pieces, per_block = kCopyThreads / 64;
  return static_cast<int>(std::min<int64_t>((pieces + per_block - 1) / per_block, 64 * device_cu_count()));
}

int check_caches(const int64_t* caches, int num_caches, int64_t max_page_bytes, int num_pages, Caches& c) {
  DS_REQUIRE(num_pages > 0 && num_caches >= 0 && max_page_bytes >= 0, "page and cache counts must be positive");
  DS_REQUIRE(num_caches == 0 || caches, "null cache list");
  DS_SUPPORTED(max_page_bytes <= (1 << 30) && num_caches <= 65536, "pages of at most 2^30 bytes, at most 65536 caches");
  DS_SUPPORTED(num_pages <= kMaxPages, "at most 2^31 - 2^14 - 1 pages");
  c.list = caches;
  c.count = num_caches;
  c.pieces = static_cast<int>((max_page_bytes + kPiece - 1) / kPiece);
  // copy_all numbers the pieces of a page over all caches in 32 bits.
  DS_SUPPORTED(static_cast<int64_t>(c.count) * c.pieces <= INT_MAX, "at most 2^43 bytes per page over all caches");
  return DS_OK;
}

int check_table(int32_t* table, int64_t stride, int rows, int width, const int32_t* refs, int num_pages, Table& t) {
  DS_REQUIRE(num_pages > 0 && rows >= 0 && width >= 0, "page, row and column counts must be positive");
  DS_REQUIRE(refs && (table || rows == 0 || width == 0), "null tensor pointer");
  DS_REQUIRE(stride >= width || rows <= 1, "block table rows overlap");
  DS_SUPPORTED(rows <= kMaxList, "at most %d block table rows", kMaxList);
  DS_SUPPORTED(num_pages <= kMaxPages, "at most 2^31 - 2^14 - 1 pages");
  // The pages that an extension needs are counted in 32 bits.
  DS_SUPPORTED(static_cast<int64_t>(rows) * width <= INT_MAX, "at most 2^31 - 1 block table entries");
  t = {table, stride, rows, width};
  return DS_OK;
}

int check_list(int count, int block_size) {
  DS_REQUIRE(count >= 0 && block_size > 0, "counts and the page size must be positive");
  DS_SUPPORTED(count <= kMaxList, "at most %d rows per call", kMaxList);
  return DS_OK;
}

size_t workspace_bytes(int num_pages) {
  if (num_pages <= 0) return 0;
  return sizeof(int32_t) * (kHeaderWords + std::max<int64_t>(2 * static_cast<int64_t>(num_pages), kMaxList));
}

int check_workspace(const void* workspace, size_t bytes, int num_pages) {
  DS_REQUIRE(workspace && bytes >= workspace_bytes(num_pages) && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0,
             "workspace must be 16-byte aligned and hold ds_pages_workspace_bytes()");
  return DS_OK;
}

#define DS_PASS(call)              \
  do {                             \
    const int rc_ = (call);        \
    if (rc_ != DS_OK) return rc_;  \
  } while (0)

}  // namespace
}  // namespace ds355

using namespace ds355;

extern "C" size_t ds_pages_workspace_bytes(int num_pages) { return workspace_bytes(num_pages); }

extern "C" int ds_pages_copy(ds_stream_t stream, const int64_t* caches, int num_caches, int64_t max_page_bytes,
                             int num_pages, const int32_t* src, const int32_t* dst, int count, int32_t* status) {
  Caches c{};
  DS_PASS(check_caches(caches, num_caches, max_page_bytes, num_pages, c));
  DS_REQUIRE(count >= 0 && (count == 0 || (src && dst)), "null page list");
  if (count == 0 || c.count == 0 || c.pieces == 0) return clear_error();
  copy_pages_kernel<<<copy_blocks(c, count), kCopyThreads, 0, reinterpret_cast<hipStream_t>(stream)>>>(
      c, src, dst, count, num_pages, status);
  return check_launch("ds_pages_copy");
}

extern "C" int ds_pages_fork(ds_stream_t stream, const int64_t* caches, int num_caches, int64_t max_page_bytes,
                             int num_pages, int32_t* ref_counts, int32_t* block_table, int64_t bt_stride,
                             int table_rows, int table_width, const int32_t* parents, const int32_t* children,
                             const int32_t* lens, int count, int block_size, void* workspace, size_t bytes,
                             int32_t* status) {
  ForkArgs a{};
  DS_PASS(check_caches(caches, num_caches, max_page_bytes, num_pages, a.caches));
  DS_PASS(check_table(block_table, bt_stride, table_rows, table_width, ref_counts, num_pages, a.table));
  DS_PASS(check_list(count, block_size));
  DS_PASS(check_workspace(workspace, bytes, num_pages));
  if (count == 0) return clear_error();
  DS_REQUIRE(parents && children && lens, "null row list");
  a.refs = ref_counts, a.num_pages = num_pages, a.parents = parents, a.children = children, a.lens = lens;
  a.count = count, a.block_size = block_size, a.status = status;
  a.header = static_cast<int32_t*>(workspace);
  a.page = a.header + kHeaderWords;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  fork_release_kernel<<<count, kThreadsP, 0, s>>>(a);
  fork_share_kernel<<<count + copy_blocks(a.caches, count), kCopyThreads, 0, s>>>(a);
  return check_launch("ds_pages_fork");
}

extern "C" int ds_pages_extend(ds_stream_t stream, int num_pages, int32_t* ref_counts, int32_t* block_table,
                               int64_t bt_stride, int table_rows, int table_width, const int32_t* rows,
                               const int32_t* lens, int count, int block_size, int32_t* status) {
  Table t{};
  DS_PASS(check_table(block_table, bt_stride, table_rows, table_width, ref_counts, num_pages, t));
  DS_PASS(check_list(count, block_size));
  if (count == 0) return clear_error();
  DS_REQUIRE(rows && lens, "null row list");
  extend_kernel<<<1, kThreadsP, 0, reinterpret_cast<hipStream_t>(stream)>>>(t, ref_counts, num_pages, rows, lens, count,
                                                                            block_size, status);
  return check_launch("ds_pages_extend");
}

extern "C" int ds_pages_free(ds_stream_t stream, int num_pages, int32_t* ref_counts, int32_t* block_table,
                             int64_t bt_stride, int table_rows, int table_width, const int32_t* rows,
                             const int32_t* keep_lens, int count, int block_size, int32_t* status) {
  Table t{};
  DS_PASS(check_table(block_table, bt_stride, table_rows, table_width, ref_counts, num_pages, t));
  DS_PASS(check_list(count, block_size));
  if (count == 0) return clear_error();
  DS_REQUIRE(rows, "null row list");
  free_kernel<<<count, 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(t, ref_counts, num_pages, rows, keep_lens,
                                                                        block_size, status);
  return check_launch("ds_pages_free");
}

extern "C" int ds_pages_compact(ds_stream_t stream, const int64_t* caches, int num_caches, int64_t max_page_bytes,
                                int num_pages, int32_t* ref_counts, int32_t* block_table, int64_t bt_stride,
                                int table_rows, int table_width, int32_t* page_map, void* workspace, size_t bytes,
                                int32_t* status) {
  CompactArgs a{};
  DS_PASS(check_caches(caches, num_caches, max_page_bytes, num_pages, a.caches));
  DS_PASS(check_table(block_table, bt_stride, table_rows, table_width, ref_counts, num_pages, a.table));
  DS_PASS(check_workspace(workspace, bytes, num_pages));
  DS_REQUIRE(page_map, "null page map");
  a.refs = ref_counts, a.num_pages = num_pages, a.page_map = page_map, a.status = status;
  a.header = static_cast<int32_t*>(workspace);
  a.from = a.header + kHeaderWords;
  a.to = a.from + num_pages;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  compact_plan_kernel<<<1, kThreadsP, 0, s>>>(a);
  // At most half of the pages move.
  const int64_t cells = static_cast<int64_t>(table_rows) * table_width;
  const int blocks = std::max<int>(copy_blocks(a.caches, num_pages / 2),
                                   static_cast<int>(std::min<int64_t>((cells + kCopyThreads - 1) / kCopyThreads, 1024)));
  if (blocks > 0) compact_move_kernel<<<blocks, kCopyThreads, 0, s>>>(a);
  return check_launch("ds_pages_compact");
}

// RMS norm of every query and key head with the position rotation in the same pass, and the write of
// the new tokens' keys and values into the paged cache.
//
//   n = x / sqrt(mean(x^2) + eps) * w        per head, fp32
//   y = n rotated at the token's position    (a, b) -> (a c - b s, b c + a s) over rotary_dim, the rest as it is
//
// The reference's models leave this to their platform's kernels (its own rotation of gathered keys
// is diffspec/compact_kv.py:68-101, whose two pairings are used here); a verifier step needs y of the
// queries, y of the keys and the values in the target's pages, and a draft whose keys are normed
// needs n of the keys, unrotated, for its raw cache.
//
// A head is read once: a lane holds both elements of its pairs (V pairs: two V-element vectors, half
// the rotary span apart or next to each other), so the rotation needs no exchange and an output may
// take its input's place; the lanes of a head sum their squares by lane moves.  A wave keeps one
// token's cosines and sines in registers and goes through heads of it.  HBM-bound: every byte is read
// and written once.  Measured: 16411 tokens of 32 + 8 + 8 heads of 128 in bf16 with pages and normed keys,
// 446 MB, 105 us (4.24 TB/s; a large copy reaches 5.1); 16 tokens 5 us, a launch.
#include <type_traits>

#include "ds355_common.h"

namespace ds355 {
namespace {

constexpr int kThreadsQ = 256;
constexpr int32_t kStatusPosition = 1;  // a position is outside the cos/sin table
constexpr int32_t kStatusSlot = 2;      // a cache slot is outside the cache

struct Heads {  // [tokens, heads, head_dim], contiguous in head_dim; strides in elements
  void* p;
  int64_t token, head;
};

struct QkArgs {
  Heads q, k, v, q_out, k_out, n_out;
  const void* q_weight;
  const void* k_weight;
  int weight_f32;
  const void* positions;
  int positions64;
  const void* cos_sin;
  int cos_sin_f32;
  int64_t cs_stride;
  int cs_rows;
  void* key_cache;
  void* value_cache;
  int64_t kc_block, kc_token, kc_head, vc_block, vc_token, vc_head;
  const void* slots;
  int slots64;
  int block_size;
  int64_t num_slots;
  int tokens, hq, hkv, d, rot, neox;
  float eps;
  int lanes;   // lanes per head, a power of two
  int passes;  // heads that each group of lanes goes through
  int chunks;  // waves per token
  int32_t* status;
};

// V neighbouring elements as they lie in memory, widened to fp32 and rounded back (to nearest even).
// STREAM: past the caches.
template <int DT, int V>
struct Raw {
  typename Elem<DT>::T e[V];
};
template <int DT, int V, bool STREAM = false>
__device__ __forceinline__ Raw<DT, V> load_raw(const typename Elem<DT>::T* p) {
  typedef typename Elem<DT>::T T;
  Raw<DT, V> r;
  if constexpr (V == 1) {
    r.e[0] = *p;
  } else {
    constexpr int kWords = V * sizeof(T) / 4, kLoad = kWords < 4 ? kWords : 4;
    typedef uint32_t U __attribute__((ext_vector_type(kLoad)));
    uint32_t w[kWords];
#pragma unroll
    for (int i = 0; i < kWords; i += kLoad) {
      const U* from = reinterpret_cast<const U*>(reinterpret_cast<const uint32_t*>(p) + i);
      const U u = STREAM ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
      for (int k = 0; k < kLoad; ++k) w[i + k] = u[k];
    }
    __builtin_memcpy(r.e, w, sizeof(w));
  }
  return r;
}
template <int DT, int V, bool STREAM>
__device__ __forceinline__ void store_raw(typename Elem<DT>::T* p, const Raw<DT, V>& r) {
  typedef typename Elem<DT>::T T;
  if constexpr (V == 1) {
    *p = r.e[0];
  } else {
    constexpr int kWords = V * sizeof(T) / 4, kLoad = kWords < 4 ? kWords : 4;
    typedef uint32_t U __attribute__((ext_vector_type(kLoad)));
    uint32_t w[kWords];
    __builtin_memcpy(w, r.e, sizeof(w));
#pragma unroll
    for (int i = 0; i < kWords; i += kLoad) {
      U u;
#pragma unroll
      for (int k = 0; k < kLoad; ++k) u[k] = w[i + k];
      U* to = reinterpret_cast<U*>(reinterpret_cast<uint32_t*>(p) + i);
      if constexpr (STREAM) __builtin_nontemporal_store(u, to);
      else *to = u;
    }
  }
}
template <int DT, int V>
__device__ __forceinline__ void widen(const Raw<DT, V>& r, float (&x)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = Elem<DT>::load(r.e[i]);
}
template <int DT, int V, bool STREAM>
__device__ __forceinline__ void store_vec(typename Elem<DT>::T* p, const float (&x)[V]) {
  Raw<DT, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if constexpr (DT == DS_BF16) r.e[i] = __builtin_bit_cast(uint16_t, static_cast<__bf16>(x[i]));
    else r.e[i] = Elem<DT>::store(x[i]);
  }
  store_raw<DT, V, STREAM>(p, r);
}
template <int DT, int V>
__device__ __forceinline__ void load_any(const void* p, bool f32, int64_t at, float (&x)[V]) {
  if (f32) widen<DS_FP32, V>(load_raw<DS_FP32, V>(static_cast<const float*>(p) + at), x);
  else widen<DT, V>(load_raw<DT, V>(static_cast<const typename Elem<DT>::T*>(p) + at), x);
}

__device__ __forceinline__ int64_t index_at(const void* p, int is64, int t) {
  return is64 ? static_cast<const int64_t*>(p)[t] : static_cast<int64_t>(static_cast<const int32_t*>(p)[t]);
}

// A lane's pairs: item i of a head is V pairs, elements `a` .. a + V - 1 and `b` .. b + V - 1.  Items
// past the rotary span are two neighbouring vectors that only the norm touches.
struct Item {
  int a, b, pair;  // pair: first cosine, or -1
  bool on;
};
template <int V, bool NEOX>
__device__ __forceinline__ Item item_at(const QkArgs& g, int i) {
  Item it;
  const int turned = g.rot / (2 * V);
  it.on = i < g.d / (2 * V);
  it.pair = i < turned ? i * V : -1;
  const bool apart = NEOX && i < turned;
  it.a = apart ? i * V : 2 * i * V;
  it.b = apart ? g.rot / 2 + i * V : it.a + V;
  if (!it.on) it.a = it.b = 0;
  return it;
}

template <int DT, int V, int NI, bool NEOX, bool STREAM>
__global__ __launch_bounds__(kThreadsQ) void qk_norm_rope_kernel(QkArgs g) {
  typedef typename Elem<DT>::T T;
  const int lane = threadIdx.x & 63;
  const int wave = blockIdx.x * (kThreadsQ / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int token = wave / g.chunks, chunk = wave - token * g.chunks;
  if (token >= g.tokens) return;
  const int groups = 64 / g.lanes, group = lane / g.lanes, in_head = lane & (g.lanes - 1);
  const int heads = g.hq + g.hkv + (g.value_cache ? g.hkv : 0);
  Item it[NI];
#pragma unroll
  for (int n = 0; n < NI; ++n) it[n] = item_at<V, NEOX>(g, in_head + n * g.lanes);
  // A head's elements as they lie in memory; the next pass's are on their way while one is worked on.
  Raw<DT, V> ra[NI], rb[NI];
  auto fetch = [&](int pass) {
    const int head = (chunk * g.passes + pass) * groups + group;
    if (pass >= g.passes || head >= heads) return;
    const bool is_q = head < g.hq, is_v = head >= g.hq + g.hkv;
    const T* x = static_cast<const T*>(is_q ? g.q.p : is_v ? g.v.p : g.k.p) + token * (is_q ? g.q.token : is_v ? g.v.token : g.k.token) +
                 (is_q ? head * g.q.head : is_v ? (head - g.hq - g.hkv) * g.v.head : (head - g.hq) * g.k.head);
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      if (!it[n].on) continue;
      ra[n] = load_raw<DT, V, STREAM>(x + it[n].a);
      rb[n] = load_raw<DT, V, STREAM>(x + it[n].b);
    }
  };
  fetch(0);
  const int64_t position = index_at(g.positions, g.positions64, token);
  int64_t key_at = -1, value_at = 0;
  if (g.slots) {
    const int64_t slot = index_at(g.slots, g.slots64, token);
    if (slot >= g.num_slots) {
      if (chunk == 0 && lane == 0 && g.status) {
        __hip_atomic_fetch_or(g.status, kStatusSlot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    } else if (slot >= 0) {
      const uint32_t block = static_cast<uint32_t>(slot) / static_cast<uint32_t>(g.block_size);
      const uint32_t in = static_cast<uint32_t>(slot) - block * static_cast<uint32_t>(g.block_size);
      key_at = block * g.kc_block + in * g.kc_token;
      value_at = block * g.vc_block + in * g.vc_token;
    }
  }
  if (g.rot > 0 && (position < 0 || position >= g.cs_rows)) {  // without a rotation no row of the table is read
    if (chunk == 0 && lane == 0 && g.status) {
      __hip_atomic_fetch_or(g.status, kStatusPosition, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    return;
  }
  float c[NI][V], s[NI][V];
#pragma unroll
  for (int n = 0; n < NI; ++n) {
#pragma unroll
    for (int i = 0; i < V; ++i) c[n][i] = 1.f, s[n][i] = 0.f;
    if (it[n].on && it[n].pair >= 0) {
      load_any<DT, V>(g.cos_sin, g.cos_sin_f32, position * g.cs_stride + it[n].pair, c[n]);
      load_any<DT, V>(g.cos_sin, g.cos_sin_f32, position * g.cs_stride + g.rot / 2 + it[n].pair, s[n]);
    }
  }
  const float inv_d = 1.f / static_cast<float>(g.d);
  for (int pass = 0; pass < g.passes; ++pass) {
    const int head = (chunk * g.passes + pass) * groups + group;
    const bool on = head < heads;
    const bool is_q = head < g.hq, is_v = head >= g.hq + g.hkv;
    const int h = is_q ? head : is_v ? head - g.hq - g.hkv : head - g.hq;
    if (on && is_v && key_at >= 0) {
      T* to = static_cast<T*>(g.value_cache) + value_at + h * g.vc_head;
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        if (!it[n].on) continue;
        store_raw<DT, V, STREAM>(to + it[n].a, ra[n]);
        store_raw<DT, V, STREAM>(to + it[n].b, rb[n]);
      }
    }
    float a[NI][V], b[NI][V], sum = 0.f;
#pragma unroll
    for (int n = 0; n < NI; ++n) {
#pragma unroll
      for (int i = 0; i < V; ++i) a[n][i] = b[n][i] = 0.f;
      if (on && it[n].on) {
        widen<DT, V>(ra[n], a[n]);
        widen<DT, V>(rb[n], b[n]);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) sum += a[n][i] * a[n][i] + b[n][i] * b[n][i];
    }
    fetch(pass + 1);
    for (int off = g.lanes >> 1; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if (!on || is_v) continue;
    const float scale = 1.f / sqrtf(sum * inv_d + g.eps);
    const void* weight = is_q ? g.q_weight : g.k_weight;
    const Heads dst = is_q ? g.q_out : g.k_out;
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      if (!it[n].on) continue;
      float wa[V], wb[V];
      load_any<DT, V>(weight, g.weight_f32, it[n].a, wa);
      load_any<DT, V>(weight, g.weight_f32, it[n].b, wb);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        a[n][i] = a[n][i] * scale * wa[i];
        b[n][i] = b[n][i] * scale * wb[i];
      }
      if (!is_q && g.n_out.p) {
        T* to = static_cast<T*>(g.n_out.p) + token * g.n_out.token + h * g.n_out.head;
        store_vec<DT, V, STREAM>(to + it[n].a, a[n]);
        store_vec<DT, V, STREAM>(to + it[n].b, b[n]);
      }
      if (it[n].pair >= 0) {
        float x[2 * V], y[2 * V];
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = a[n][i], x[V + i] = b[n][i];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          // Pair i: the i-th of both halves, or the 2 i-th element and its neighbour.
          const int p = NEOX ? i : 2 * i, q = NEOX ? V + i : 2 * i + 1;
          y[p] = x[p] * c[n][i] - x[q] * s[n][i];
          y[q] = x[q] * c[n][i] + x[p] * s[n][i];
        }
#pragma unroll
        for (int i = 0; i < V; ++i) a[n][i] = y[i], b[n][i] = y[V + i];
      }
      if (dst.p) {
        T* to = static_cast<T*>(dst.p) + token * dst.token + h * dst.head;
        store_vec<DT, V, STREAM>(to + it[n].a, a[n]);
        store_vec<DT, V, STREAM>(to + it[n].b, b[n]);
      }
      if (!is_q && key_at >= 0) {
        T* to = static_cast<T*>(g.key_cache) + key_at + h * g.kc_head;
        store_vec<DT, V, STREAM>(to + it[n].a, a[n]);
        store_vec<DT, V, STREAM>(to + it[n].b, b[n]);
      }
    }
  }
}

template <int DT, int V, int NI>
int launch(hipStream_t stream, QkArgs& g) {
  const int items = g.d / (2 * V);
  g.lanes = 1;
  while (g.lanes < items && g.lanes < 64) g.lanes *= 2;
  const int heads = g.hq + g.hkv + (g.value_cache ? g.hkv : 0);
  const int rounds = (heads + 64 / g.lanes - 1) / (64 / g.lanes);  // passes of one wave over a token
  // Few tokens: a wave per pass, as many as there are; many: a wave keeps its cosines for up to 8 passes.
  const int64_t waves = static_cast<int64_t>(g.tokens) * rounds;
  g.passes = static_cast<int>(std::min<int64_t>(std::min(rounds, 8), std::max<int64_t>(1, waves / 8192)));
  g.chunks = (rounds + g.passes - 1) / g.passes;
  const int64_t total = static_cast<int64_t>(g.tokens) * g.chunks;
  const int64_t blocks = (total + kThreadsQ / 64 - 1) / (kThreadsQ / 64);
  DS_SUPPORTED(total < INT_MAX, "too many tokens and heads for one launch");
  // Heads that the 32 MiB of L2 cannot hold anyway do not pass through it: 16411 tokens of 32 + 8 heads of
  // 128 with all outputs 105.8 us, else 112.9; without normed keys 192 MiB of heads 99.4, else 106.1, but 48 MiB
  // 28.4, else 24.3, and 35 MiB 22.3, else 21.3.  With the attention that reads them next the two ways are
  // alike: 1653 and 1654, 238.7 and 236.6, 567.3 and 566.7.
  auto run = [&](auto neox, auto streamed) {
    qk_norm_rope_kernel<DT, V, NI, neox.value, streamed.value>
        <<<static_cast<unsigned>(blocks), kThreadsQ, 0, stream>>>(g);
  };
  const int64_t bytes = static_cast<int64_t>(g.tokens) * heads * g.d * sizeof(typename Elem<DT>::T);
  if (V == 8 && bytes > (int64_t{32} << 20)) {
    constexpr std::bool_constant<V == 8> kStream{};
    if (g.neox) run(std::true_type{}, kStream);
    else run(std::false_type{}, kStream);
  } else if (g.neox) {
    run(std::true_type{}, std::false_type{});
  } else {
    run(std::false_type{}, std::false_type{});
  }
  return check_launch("ds_qk_norm_rope");
}

// Vectors of V elements cover the head: pairs, the part past the rotary span, strides and addresses.
bool covers(const QkArgs& g, int size, int v) {
  if (g.d % (2 * v) || (g.neox ? (g.rot / 2) % v : g.rot % (2 * v)) || (g.d - g.rot) % (2 * v)) return false;
  const Heads all[] = {g.q, g.k, g.v, g.q_out, g.k_out, g.n_out,
                       {g.key_cache, g.kc_block | g.kc_token, g.kc_head},
                       {g.value_cache, g.vc_block | g.vc_token, g.vc_head}};
  for (const Heads& h : all) {
    if (h.p && (reinterpret_cast<uintptr_t>(h.p) % (size * v) || h.token % v || h.head % v)) return false;
  }
  const int weight = g.weight_f32 ? 4 : size, table = g.cos_sin_f32 ? 4 : size;
  return reinterpret_cast<uintptr_t>(g.q_weight) % (weight * v) == 0 &&
         reinterpret_cast<uintptr_t>(g.k_weight) % (weight * v) == 0 &&
         (g.rot == 0 || (reinterpret_cast<uintptr_t>(g.cos_sin) % (table * v) == 0 && g.cs_stride % v == 0 &&
                         (g.rot / 2) % v == 0));
}

template <int DT>
int launch_type(hipStream_t stream, QkArgs& g) {
  constexpr int kSize = DT == DS_FP32 ? 4 : 2;
  if constexpr (kSize == 2) {
    if (covers(g, kSize, 8)) return launch<DT, 8, 1>(stream, g);
  }
  if (covers(g, kSize, 4)) return launch<DT, 4, 1>(stream, g);
  return launch<DT, 1, 2>(stream, g);
}

int qk_impl(hipStream_t stream, const ds_qk_norm_rope_desc* d) {
  DS_REQUIRE(d != nullptr, "null descriptor");
  DS_REQUIRE(d->dtype == DS_BF16 || d->dtype == DS_FP16 || d->dtype == DS_FP32, "tensors must use BF16, FP16 or FP32");
  DS_REQUIRE(d->weight_dtype == d->dtype || d->weight_dtype == DS_FP32, "weights must use the tensors' dtype or FP32");
  DS_REQUIRE(d->cos_sin_dtype == d->dtype || d->cos_sin_dtype == DS_FP32,
             "the cos/sin cache must use the tensors' dtype or FP32");
  DS_REQUIRE(d->tokens >= 0 && d->num_q_heads > 0 && d->num_kv_heads > 0, "token and head counts must be positive");
  DS_REQUIRE(d->head_dim > 0 && d->head_dim % 2 == 0, "head_dim must be even");
  DS_SUPPORTED(d->head_dim <= 256, "head_dim must be at most 256");
  DS_REQUIRE(d->rotary_dim >= 0 && d->rotary_dim <= d->head_dim && d->rotary_dim % 2 == 0,
             "rotary_dim must be even and between zero and head_dim");
  DS_REQUIRE(d->cs_rows >= 0 && (d->cs_rows <= 1 || d->cs_stride >= d->rotary_dim),
             "cos/sin cache rows must hold rotary_dim values");
  if (d->tokens == 0) return clear_error();
  const bool paged = d->key_cache || d->value_cache || d->slot_mapping;
  DS_REQUIRE(!paged || (d->key_cache && d->value_cache && d->slot_mapping && d->value),
             "the paged write needs key_cache, value_cache, slot_mapping and value together");
  DS_REQUIRE(!paged || (d->block_size > 0 && d->num_blocks > 0), "page sizes and counts must be positive");
  DS_SUPPORTED(!paged || static_cast<int64_t>(d->num_blocks) * d->block_size <= INT_MAX, "at most 2^31 - 1 cache slots");
  DS_REQUIRE(d->query && d->key && d->q_weight && d->k_weight && d->positions && d->query_out &&
                 (d->cos_sin || d->rotary_dim == 0),
             "null tensor pointer");
  QkArgs g{};
  g.q = {const_cast<void*>(d->query), d->q_row_stride, d->q_head_stride};
  g.k = {const_cast<void*>(d->key), d->k_row_stride, d->k_head_stride};
  g.v = {const_cast<void*>(paged ? d->value : nullptr), d->v_row_stride, d->v_head_stride};
  g.q_out = {d->query_out, d->qo_row_stride, d->qo_head_stride};
  g.k_out = {d->key_out, d->ko_row_stride, d->ko_head_stride};
  g.n_out = {d->normed_key, d->nk_row_stride, d->nk_head_stride};
  g.q_weight = d->q_weight;
  g.k_weight = d->k_weight;
  g.weight_f32 = d->weight_dtype == DS_FP32;
  g.positions = d->positions;
  g.positions64 = d->positions_int64;
  g.cos_sin = d->cos_sin;
  g.cos_sin_f32 = d->cos_sin_dtype == DS_FP32;
  g.cs_stride = d->cs_stride;
  g.cs_rows = d->cs_rows;
  if (paged) {
    g.key_cache = d->key_cache;
    g.value_cache = d->value_cache;
    g.kc_block = d->kc_block_stride, g.kc_token = d->kc_token_stride, g.kc_head = d->kc_head_stride;
    g.vc_block = d->vc_block_stride, g.vc_token = d->vc_token_stride, g.vc_head = d->vc_head_stride;
    g.slots = d->slot_mapping;
    g.slots64 = d->slots_int64;
    g.block_size = d->block_size;
    g.num_slots = static_cast<int64_t>(d->num_blocks) * d->block_size;
  }
  g.tokens = d->tokens, g.hq = d->num_q_heads, g.hkv = d->num_kv_heads, g.d = d->head_dim, g.rot = d->rotary_dim;
  g.neox = d->is_neox_style ? 1 : 0;
  g.eps = d->eps;
  g.status = d->status;
  if (d->dtype == DS_BF16) return launch_type<DS_BF16>(stream, g);
  if (d->dtype == DS_FP16) return launch_type<DS_FP16>(stream, g);
  return launch_type<DS_FP32>(stream, g);
}

}  // namespace
}  // namespace ds355

extern "C" int ds_qk_norm_rope(ds_stream_t stream, const ds_qk_norm_rope_desc* desc) {
  return ds355::qk_impl(reinterpret_cast<hipStream_t>(stream), desc);
}

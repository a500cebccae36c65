// Writing the paged cache: tokens' keys and values appended, with the norms
// and the position rotation on the way, and the rows of accepted tokens moved
// together.

#include "paged_cache.h"

namespace tjk {

int check_cache(const char* who, const tjk_paged_cache* c, bool writes) {
  if (!c || !c->k || !c->v) return fail(TJK_EINVAL, "%s: null cache", who);
  if (c->dtype != TJK_F16 && c->dtype != TJK_BF16) return fail(TJK_EINVAL, "%s: bad cache dtype %d", who, c->dtype);
  if (c->kv_heads <= 0 || c->pages <= 0 || c->head_dim <= 0)
    return fail(TJK_EINVAL, "%s: bad cache shape pages=%lld kv_heads=%d head_dim=%d", who, (long long)c->pages, c->kv_heads,
                c->head_dim);
  if (c->head_dim % 16 || c->head_dim > 128)
    return fail(TJK_EUNSUPPORTED, "%s: head_dim=%d must be a multiple of 16 and <= 128", who, c->head_dim);
  if (c->page_size < 16 || c->page_size > 65536 || (c->page_size & (c->page_size - 1)))
    return fail(TJK_EUNSUPPORTED, "%s: page_size=%d must be a power of two from 16 to 65536", who, c->page_size);
  if (c->pages > INT32_MAX / c->page_size) return fail(TJK_EUNSUPPORTED, "%s: the cache's rows exceed int32", who);
  if (c->page_stride < 0 || c->head_stride < 0 || c->row_stride < c->head_dim)
    return fail(TJK_EINVAL, "%s: bad cache strides", who);
  if (writes && ((c->pages > 1 && c->page_stride < c->head_dim) || (c->kv_heads > 1 && c->head_stride < c->head_dim)))
    return fail(TJK_EINVAL, "%s: rows of the cache overlap", who);
  if (c->page_stride % 8 || c->head_stride % 8 || c->row_stride % 8)
    return fail(TJK_EUNSUPPORTED, "%s: cache strides must be multiples of 8", who);
  if (c->row_stride > 1 << 20 || c->row_stride * c->page_size > 1 << 29)
    return fail(TJK_EUNSUPPORTED, "%s: cache row stride %lld is too large", who, (long long)c->row_stride);
  if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return fail(TJK_EUNSUPPORTED, "%s: misaligned cache", who);
  return TJK_OK;
}

int check_written(const char* who, const tjk_paged_cache* c, int layers, int64_t layer_stride) {
  const StridedRows rows = StridedRows(c->k, 2 * c->head_dim)
                               .by(2 * c->page_stride, c->pages)
                               .by(2 * c->head_stride, c->kv_heads)
                               .by(2 * c->row_stride, c->page_size)
                               .by(2 * layer_stride, layers);
  if (rows_overlap(rows)) return fail(TJK_EINVAL, "%s: rows of the cache overlap", who);
  return TJK_OK;
}

// ------------------------------------------------------------- append
//
// One head of one token belongs to G neighbouring lanes (G the power of two from
// head_dim / 16 up); each holds two 8-element pieces, those that the rotation
// brings together: pieces p and p + rot / 16 of the halves' form (element i
// turns with i + rot / 2), and past the rotated ones neighbours.  The norm sums
// over the G lanes.  A wave takes 64 / G heads of one token.
//
// Bound by memory: 65536 tokens of 16 + 2 x 16 heads of 64 with norms, bf16, 157 us,
// 5.2 TB/s (a copy of 1 GB: 5.1); 4096 tokens of 32 + 2 x 8 heads of 128 22.3 us, 4.6; 1003
// of them 6.2 to 7.0 us.  8 tokens: 3.3 to 4 us, a launch and two passages of memory (position and
// row, then the angles).

struct AppendArgs {
  const char* qkv;
  int64_t token_bytes, head_bytes;
  const int32_t* positions;
  const float* table;
  int n_positions;
  int rot8;  // rotated pieces
  char* q_out;
  int64_t q_token_bytes, q_head_bytes;
  char* k_out;
  int64_t k_token_bytes, k_head_bytes;
  Paged cache;
  const int32_t* slots;
  const float* q_gamma;
  const float* k_gamma;
  float eps;
  int* index_errors;
  int64_t tokens;
  int heads, kv_heads, hd8;  // hd8: pieces of a head
};

// Sum over groups of G lanes (G <= 8, a power of two), in each of them.
template <int G>
__device__ __forceinline__ float group_sum(float v) {
  if constexpr (G >= 2)
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true));
  if constexpr (G >= 4)
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, true));
  if constexpr (G >= 8)
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x141, 0xF, 0xF, true));
  return v;
}

template <typename T, int G, bool INTER>
__global__ __launch_bounds__(256) void rope_append_kernel(AppendArgs a) {
  constexpr int HPW = 64 / G;  // heads of a wave
  const int lane = threadIdx.x & 63, g = lane / G, p = lane % G;
  const int all = a.heads + 2 * a.kv_heads;
  const uint32_t blocks = (uint32_t)(all + HPW - 1) / HPW;
  const uint32_t wave = blockIdx.x * 4 + (threadIdx.x >> 6), tok = wave / blocks;
  const int h = (int)(wave - tok * blocks) * HPW + g;
  if ((int)tok >= a.tokens) return;
  const int64_t t = tok;
  const int pos = a.positions[t];
  const int slot = a.slots ? a.slots[t] : -1;
  const bool in = h < all && 2 * p < a.hd8;
  const int half = a.rot8 >> 1;
  const bool turned = p < half;
  const int c0 = !in ? 0 : turned && !INTER ? p : 2 * p, c1 = !in ? 0 : turned && !INTER ? p + half : 2 * p + 1;

  // every load goes out before the first is waited for, but for the angles, which
  // lie where the position says
  const T* const src = reinterpret_cast<const T*>(a.qkv + t * a.token_bytes + (int64_t)(in ? h : 0) * a.head_bytes);
  const typename Oct<T>::raw r0 = Oct<T>::load(src + 8 * c0), r1 = Oct<T>::load(src + 8 * c1);
  const float* const gamma = h < a.heads ? a.q_gamma : h < a.heads + a.kv_heads ? a.k_gamma : nullptr;
  Oct<float>::raw g0{}, g1{};
  if (gamma) {
    g0 = Oct<float>::load(gamma + 8 * c0);
    g1 = Oct<float>::load(gamma + 8 * c1);
  }
  const bool placed = pos >= 0 && pos < a.n_positions;
  const bool stored = placed && slot >= 0 && (slot >> a.cache.shift) < a.cache.pages;
  const bool turns = in && turned && placed && h < a.heads + a.kv_heads;
  Oct<float>::raw w0{}, w1{};
  if (turns) {
    const float* const cs = a.table + ((int64_t)pos * (4 * a.rot8) + 8 * p) * 2;
    w0 = Oct<float>::load(cs);
    w1 = Oct<float>::load(cs + 8);
  }
  if (h == 0 && p == 0 && a.index_errors && (!placed || (slot >= 0 && !stored))) atomicAdd(a.index_errors, 1);

  float x[2][8];
  Oct<T>::to(r0, x[0]);
  Oct<T>::to(r1, x[1]);
  float sum = 0.f;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(x[u][i], x[u][i], sum);
  sum = group_sum<G>(in ? sum : 0.f);
  if (gamma) {
    const float r = 1.0f / sqrtf(sum / (float)(8 * a.hd8) + a.eps);
    float f[2][8];
    Oct<float>::to(g0, f[0]);
    Oct<float>::to(g1, f[1]);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) x[u][i] *= r * f[u][i];
  }
  if (turns) {
    float w[2][8];
    Oct<float>::to(w0, w[0]);
    Oct<float>::to(w1, w[1]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // the pair's members: element i of both pieces, or elements 2 j, 2 j + 1 of one
      float &u = INTER ? x[i >> 2][2 * (i & 3)] : x[0][i], &v = INTER ? x[i >> 2][2 * (i & 3) + 1] : x[1][i];
      const float c = w[i >> 2][2 * (i & 3)], s = w[i >> 2][2 * (i & 3) + 1];
      const float y = u * c - v * s;
      v = v * c + u * s;
      u = y;
    }
  }
  if (!in) return;
  if (!placed) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[0][i] = x[1][i] = 0.f;
  }
  auto put = [&](char* row) {
    reinterpret_cast<uint4*>(row)[c0] = Oct<T>::from(x[0]);
    reinterpret_cast<uint4*>(row)[c1] = Oct<T>::from(x[1]);
  };
  if (h < a.heads) {
    put(a.q_out + t * a.q_token_bytes + h * a.q_head_bytes);
    return;
  }
  const bool key = h < a.heads + a.kv_heads;
  const int kh = key ? h - a.heads : h - a.heads - a.kv_heads;
  if (key && a.k_out) put(a.k_out + t * a.k_token_bytes + kh * a.k_head_bytes);
  if (stored)
    put((key ? a.cache.k : a.cache.v) + (int64_t)(slot >> a.cache.shift) * a.cache.page_bytes + kh * a.cache.head_bytes +
        (int64_t)(slot & ((1 << a.cache.shift) - 1)) * a.cache.row_bytes);
}

// ------------------------------------------------------------ compaction
//
// A wave moves the keys and the values of one (layer, sequence, head), a lane one
// 16-byte piece of a row: the places first, then the loads, then the stores.  Row
// path[i] >= i goes to row i, so no row is overwritten before it is read.
//
// Bound by latency (counts and path, places, rows: three passages of memory one
// after the other), then by memory, which does not like 256 bytes here and 256
// there: 24 layers x 64 sequences x 8 heads of 128, 7 rows each, 25.5 us, 3.7 TB/s read
// and written (21.5 on the same rows again); four layers of 8 sequences 3.6 us.  Where
// this took 27 and 5, keys and values in waves of their own took 29 and 6 us, two
// instructions of rows in flight instead of four 28.5 and 4.4.
// Loads where nothing moves, from one place for all, to spare the lanes' conditions:
// 40 and 13.

struct CompactArgs {
  Paged cache;
  int64_t layer_bytes;
  const int32_t* table;
  int64_t ld_table;
  int table_cols;
  const int32_t* ctx_lens;
  const int32_t* path;
  int64_t ld_path;
  int max_nodes;
  const int32_t* count;
  int* index_errors;
  int layers, batch, kv_heads, hd8;
};

template <int CPR>  // lanes per row
__global__ __launch_bounds__(256) void compact_kernel(CompactArgs a) {
  constexpr int RPI = 64 / CPR, U = 4;  // rows of an instruction, instructions in flight
  const int lane = threadIdx.x & 63, r = lane / CPR, c = lane % CPR;
  const uint32_t wave = blockIdx.x * 4 + (threadIdx.x >> 6), lb = wave / (uint32_t)a.kv_heads;
  const int h = (int)(wave - lb * a.kv_heads), layer = (int)(lb / (uint32_t)a.batch), b = (int)(lb - layer * a.batch);
  if (layer >= a.layers) return;
  char* const kb = a.cache.k + layer * a.layer_bytes + h * a.cache.head_bytes;
  char* const vb = a.cache.v + layer * a.layer_bytes + h * a.cache.head_bytes;
  const int n = min(a.count[b], a.max_nodes);
  const int64_t ctx = max(a.ctx_lens[b], 0);
  const int32_t* const row = a.table + b * a.ld_table;
  const int32_t* const path = a.path + b * a.ld_path;
  const int64_t room = (int64_t)a.table_cols << a.cache.shift;
  const int mask = (1 << a.cache.shift) - 1;
  for (int i0 = 1; i0 < n; i0 += U * RPI) {
    int64_t src[U], dst[U];
    int from[U], ps[U], pd[U];
    bool named[U], moves[U], lost = false;
#pragma unroll
    for (int u = 0; u < U; ++u) from[u] = path[min(i0 + u * RPI + r, a.max_nodes - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * RPI + r;
      named[u] = i < n && from[u] >= i && from[u] < a.max_nodes && ctx + from[u] < room;  // (and ctx + i, which is less)
      ps[u] = page_of(row, named[u] ? (int)((ctx + from[u]) >> a.cache.shift) : 0, a.cache.pages);
      pd[u] = page_of(row, named[u] ? (int)((ctx + i) >> a.cache.shift) : 0, a.cache.pages);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * RPI + r;
      const bool there = named[u] && ps[u] >= 0 && pd[u] >= 0;
      moves[u] = there && c < a.hd8;
      lost |= i < n && !there;
      src[u] = ps[u] * a.cache.page_bytes + ((ctx + from[u]) & mask) * a.cache.row_bytes + 16 * c;
      dst[u] = pd[u] * a.cache.page_bytes + ((ctx + i) & mask) * a.cache.row_bytes + 16 * c;
    }
    uint4 k[U], v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      k[u] = v[u] = make_uint4(0, 0, 0, 0);
      if (moves[u]) {
        k[u] = *reinterpret_cast<const uint4*>(kb + src[u]);
        v[u] = *reinterpret_cast<const uint4*>(vb + src[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (moves[u]) {
        *reinterpret_cast<uint4*>(kb + dst[u]) = k[u];
        *reinterpret_cast<uint4*>(vb + dst[u]) = v[u];
      }
    if (lost && layer == 0 && h == 0 && c == 0 && a.index_errors) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * RPI + r < n && !moves[u]) atomicAdd(a.index_errors, 1);
    }
  }
}

}  // namespace tjk

using namespace tjk;

extern "C" int tjk_rope_append(const void* qkv, int64_t ld_token, int64_t ld_head, const int32_t* positions,
                               const float* table, int64_t n_positions, int64_t rot, int interleaved, void* q_out,
                               int64_t ld_q_token, int64_t ld_q_head, void* k_out, int64_t ld_k_token, int64_t ld_k_head,
                               const tjk_paged_cache* cache, const int32_t* slots, const float* q_gamma,
                               const float* k_gamma, float eps, int* index_errors, int64_t tokens, int heads, int kv_heads,
                               int head_dim, int dtype, void* stream) {
  const char* const who = "tjk_rope_append";
  if (tokens < 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || n_positions < 0 || rot < 0)
    return fail(TJK_EINVAL, "%s: bad shape tokens=%lld heads=%d kv_heads=%d head_dim=%d", who, (long long)tokens, heads,
                kv_heads, head_dim);
  if (dtype != TJK_F16 && dtype != TJK_BF16) return fail(TJK_EINVAL, "%s: bad dtype %d", who, dtype);
  if (head_dim % 16 || head_dim > 128)
    return fail(TJK_EUNSUPPORTED, "%s: head_dim=%d must be a multiple of 16 and <= 128", who, head_dim);
  if (rot % 16 || rot > head_dim)
    return fail(TJK_EUNSUPPORTED, "%s: %lld rotated elements must be a multiple of 16 and <= head_dim", who, (long long)rot);
  if (heads > 65536 || kv_heads > 65536 || tokens > INT32_MAX || n_positions > INT32_MAX)
    return fail(TJK_EUNSUPPORTED, "%s: too large", who);
  if (cache) {
    if (const int bad = check_cache(who, cache, true)) return bad;
    if (cache->dtype != dtype || cache->kv_heads != kv_heads || cache->head_dim != head_dim)
      return fail(TJK_EINVAL, "%s: the cache's dtype, heads or head_dim differ", who);
  }
  if (tokens == 0) return TJK_OK;
  if (!qkv || !positions || !q_out || (rot > 0 && !table) || (!cache != !slots))
    return fail(TJK_EINVAL, "%s: null pointer", who);
  if (ld_head < head_dim || ld_q_head < head_dim || (k_out && ld_k_head < head_dim) || ld_token < 0 || ld_q_token < 0 ||
      (k_out && ld_k_token < 0))
    return fail(TJK_EINVAL, "%s: stride too small", who);
  if (ld_token % 8 || ld_head % 8 || ld_q_token % 8 || ld_q_head % 8 || (k_out && (ld_k_token % 8 || ld_k_head % 8)))
    return fail(TJK_EUNSUPPORTED, "%s: strides must be multiples of 8", who);
  if (tokens > 1 && (ld_q_token < head_dim || (k_out && ld_k_token < head_dim)))
    return fail(TJK_EINVAL, "%s: a stride too small for a row of its own", who);
  if ((((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)table | (uintptr_t)q_gamma | (uintptr_t)k_gamma) & 15))
    return fail(TJK_EUNSUPPORTED, "%s: misaligned pointer", who);
  // a lane writes what it has read, as long as it lies in the same place (a stride of
  // which there is one step only says nothing)
  const char* const keys = static_cast<const char*>(qkv) + 2 * heads * ld_head;
  auto elsewhere = [&](int64_t token, int64_t head, int rows) {
    return (tokens > 1 && token != ld_token) || (rows > 1 && head != ld_head);
  };
  if ((q_out == qkv && elsewhere(ld_q_token, ld_q_head, heads)) ||
      (k_out && ((k_out == keys && elsewhere(ld_k_token, ld_k_head, kv_heads)) || k_out == qkv)))
    return fail(TJK_EINVAL, "%s: outputs may alias qkv only in place", who);
  auto rows = [&](const void* base, int64_t token, int64_t head, int n) {
    return StridedRows(base, 2 * head_dim).by(2 * token, tokens).by(2 * head, n);
  };
  const StridedRows in = rows(qkv, ld_token, ld_head, heads + 2 * kv_heads), q_rows = rows(q_out, ld_q_token, ld_q_head, heads),
                    k_rows = rows(k_out, ld_k_token, ld_k_head, kv_heads);
  if (rows_overlap(q_rows) || (k_out && rows_overlap(k_rows))) return fail(TJK_EINVAL, "%s: rows of an output overlap", who);
  const bool in_place = q_out == qkv || (k_out && k_out == keys);
  if ((q_out != qkv && rows_meet(q_rows, in)) || (k_out && k_out != keys && rows_meet(k_rows, in)) || (in_place && rows_overlap(in)))
    return fail(TJK_EINVAL, "%s: outputs may overlap qkv only in place", who);
  if (k_out && rows_meet(q_rows, k_rows)) return fail(TJK_EINVAL, "%s: q_out and k_out overlap", who);
  if (cache) {
    if (const int bad = check_written(who, cache, 1, 0)) return bad;
    auto page = [&](const void* base) {
      return StridedRows(base, 2 * head_dim).by(2 * cache->head_stride, kv_heads).by(2 * cache->row_stride, cache->page_size);
    };
    if (rows_meet(page(cache->k), page(cache->v))) return fail(TJK_EINVAL, "%s: a page's keys and values overlap", who);
  }
  AppendArgs a{static_cast<const char*>(qkv), 2 * ld_token, 2 * ld_head, positions, table, (int)n_positions, (int)rot / 8,
               static_cast<char*>(q_out), 2 * ld_q_token, 2 * ld_q_head, static_cast<char*>(k_out), 2 * ld_k_token,
               2 * ld_k_head, cache ? paged(*cache) : Paged{}, slots, q_gamma, k_gamma, eps, index_errors, tokens, heads,
               kv_heads, head_dim / 8};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  auto go = [&](auto elem, auto group, auto inter) -> int {
    typedef decltype(elem) T;
    constexpr int G = decltype(group)::value;
    const int64_t blocks = (heads + 2 * (int64_t)kv_heads + 64 / G - 1) / (64 / G);
    const int64_t grid = (tokens * blocks + 3) / 4;
    if (grid > UINT32_MAX / 256 || tokens * blocks > INT32_MAX) return fail(TJK_EUNSUPPORTED, "%s: %lld tokens are too many", who, (long long)tokens);
    rope_append_kernel<T, G, decltype(inter)::value><<<(unsigned)grid, 256, 0, s>>>(a);
    return check_launch(who);
  };
  auto with_group = [&](auto elem, auto inter) -> int {
    if (head_dim <= 16) return go(elem, std::integral_constant<int, 1>{}, inter);
    if (head_dim <= 32) return go(elem, std::integral_constant<int, 2>{}, inter);
    if (head_dim <= 64) return go(elem, std::integral_constant<int, 4>{}, inter);
    return go(elem, std::integral_constant<int, 8>{}, inter);
  };
  auto with_form = [&](auto elem) -> int {
    return interleaved ? with_group(elem, std::true_type{}) : with_group(elem, std::false_type{});
  };
  return dtype == TJK_F16 ? with_form(f16(0)) : with_form(bf16(0));
}

extern "C" int tjk_compact_cache(const tjk_paged_cache* cache, int layers, int64_t layer_stride, const int32_t* block_table,
                                 int64_t ld_table, int64_t table_cols, const int32_t* ctx_lens, const int32_t* path,
                                 int64_t ld_path, int max_nodes, const int32_t* count, int* index_errors, int batch,
                                 void* stream) {
  const char* const who = "tjk_compact_cache";
  if (const int bad = check_cache(who, cache, true)) return bad;
  if (layers < 0 || batch < 0 || max_nodes < 0 || table_cols < 0)
    return fail(TJK_EINVAL, "%s: bad shape layers=%d batch=%d max_nodes=%d", who, layers, batch, max_nodes);
  if (max_nodes > 64) return fail(TJK_EUNSUPPORTED, "%s: max_nodes=%d exceeds 64", who, max_nodes);
  if (table_cols > INT32_MAX) return fail(TJK_EUNSUPPORTED, "%s: block table too wide", who);
  if (layers > 1 && (layer_stride < cache->head_dim || layer_stride % 8))
    return fail(TJK_EUNSUPPORTED, "%s: the layers' stride must be a multiple of 8 and hold a row", who);
  if (layers == 0 || batch == 0 || max_nodes < 2 || table_cols == 0) return TJK_OK;
  if (!block_table || !ctx_lens || !path || !count) return fail(TJK_EINVAL, "%s: null pointer", who);
  if (ld_table < table_cols || ld_path < max_nodes) return fail(TJK_EINVAL, "%s: leading dimension too small", who);
  if (const int bad = check_written(who, cache, layers, layer_stride)) return bad;
  const int64_t pairs = (int64_t)layers * batch, waves = pairs * cache->kv_heads;
  if (pairs > INT32_MAX || waves > INT32_MAX / 64) return fail(TJK_EUNSUPPORTED, "%s: too large", who);
  const CompactArgs a{paged(*cache), 2 * layer_stride, block_table, ld_table, (int)table_cols, ctx_lens, path, ld_path,
                      max_nodes, count, index_errors, layers, batch, cache->kv_heads, cache->head_dim / 8};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const unsigned grid = (unsigned)((waves + 3) / 4);
  auto go = [&](auto lanes) { compact_kernel<decltype(lanes)::value><<<grid, 256, 0, s>>>(a); };
  if (cache->head_dim <= 32) go(std::integral_constant<int, 4>{});
  else if (cache->head_dim <= 64) go(std::integral_constant<int, 8>{});
  else go(std::integral_constant<int, 16>{});
  return check_launch(who);
}

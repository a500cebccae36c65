// Attention of drafted tokens over the paged cache.
//
// A sequence has c tokens behind it, whose keys and values are positions 0 ..
// c - 1 of its pages, and n <= 64 nodes (drafted tokens, parents first) at
// positions c .. c + n - 1.  A node sees all of the c tokens and the nodes that
// its mask names.  Query head h reads key head h / (heads / kv_heads).

#include "paged_cache.h"

namespace tjk {

struct TreeArgs {
  const char* q;
  int64_t q_token_bytes, q_head_bytes;
  Paged cache;
  const int32_t* table;
  int64_t ld_table;
  int table_cols;
  const int32_t* ctx_lens;
  const int32_t* cu_nodes;
  const uint64_t* mask;
  char* out;
  int64_t out_bytes;  // of a row
  float scale;
  int* index_errors;
  int64_t tokens;
  int batch, heads, group, hd8, max_nodes;
};

// One workgroup per (sequence, head, node); a thread takes every 256th key.
template <typename T>
__global__ __launch_bounds__(256) void tree_simple_kernel(TreeArgs a) {
  __shared__ float sq[128];
  __shared__ float so[4][128 + 2];
  const int node = blockIdx.x % a.max_nodes, bh = blockIdx.x / a.max_nodes, h = bh % a.heads, b = bh / a.heads;
  const int64_t first = max(a.cu_nodes[b], 0);
  const int n = min(max(a.cu_nodes[b + 1] - a.cu_nodes[b], 0), a.max_nodes);
  const int64_t t = first + node;
  if (node >= n || t >= a.tokens) return;
  const int hd = 8 * a.hd8;
  if (threadIdx.x < hd)
    sq[threadIdx.x] = to_f32(reinterpret_cast<const T*>(a.q + t * a.q_token_bytes + h * a.q_head_bytes)[threadIdx.x]);
  __syncthreads();
  const int64_t ctx = max(a.ctx_lens[b], 0);
  const int64_t room = (int64_t)a.table_cols << a.cache.shift;
  const int64_t end = min(ctx + n, room);
  if (threadIdx.x == 0 && node == 0 && end < ctx + n && a.index_errors) atomicAdd(a.index_errors, 1);
  const uint64_t bits = a.mask ? a.mask[t] : ~0ull >> (63 - node);
  const int32_t* const row = a.table + b * a.ld_table;
  const int64_t head = (h / a.group) * a.cache.head_bytes;
  float m = -INFINITY, l = 0.f, o[128];
#pragma unroll
  for (int i = 0; i < 128; ++i) o[i] = 0.f;
  for (int64_t x = threadIdx.x; x < end; x += 256) {
    if (x >= ctx && !(bits >> (x - ctx) & 1)) continue;
    const int pg = page_of(row, (int)(x >> a.cache.shift), a.cache.pages);
    if (pg < 0) {
      if (node == 0 && a.index_errors) atomicAdd(a.index_errors, 1);
      continue;
    }
    const int64_t at = pg * a.cache.page_bytes + head + (x & ((1 << a.cache.shift) - 1)) * (int64_t)a.cache.row_bytes;
    float s = 0.f;
    for (int c = 0; c < a.hd8; ++c) {
      float k[8];
      Oct<T>::to(Oct<T>::load(reinterpret_cast<const T*>(a.cache.k + at) + 8 * c), k);
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf(sq[8 * c + i], k[i], s);
    }
    s *= a.scale;
    const float m2 = fmaxf(m, s);
    if (m2 == -INFINITY) continue;
    const float keep = expf(m - m2), p = expf(s - m2);
    m = m2;
    l = l * keep + p;
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      if (c < a.hd8) {
        float v[8];
        Oct<T>::to(Oct<T>::load(reinterpret_cast<const T*>(a.cache.v + at) + 8 * c), v);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[8 * c + i] = fmaf(p, v[i], o[8 * c + i] * keep);
      }
    }
  }
  float top = m;
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  const float w = m == -INFINITY ? 0.f : expf(m - top);
  const float lw = wave_sum(l * w);
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < 128; ++i) {
    const float v = wave_sum(w == 0.f ? 0.f : o[i] * w);
    if ((threadIdx.x & 63) == 0) so[wave][i] = v;
  }
  if ((threadIdx.x & 63) == 0) so[wave][128] = top, so[wave][129] = lw;
  __syncthreads();
  if (threadIdx.x < hd) {
    float all = -INFINITY;
    for (int j = 0; j < 4; ++j) all = fmaxf(all, so[j][128]);
    float sum = 0.f, y = 0.f;
    for (int j = 0; j < 4; ++j) {
      if (so[j][128] == -INFINITY) continue;
      const float f = expf(so[j][128] - all);
      sum += f * so[j][129];
      y += f * so[j][threadIdx.x];
    }
    reinterpret_cast<T*>(a.out + t * a.out_bytes)[(int64_t)h * hd + threadIdx.x] = from_f32<T>(sum == 0.f ? 0.f : y / sum);
  }
}

}  // namespace tjk

using namespace tjk;

extern "C" size_t tjk_tree_attention_bytes(int heads, int kv_heads, int head_dim, int max_nodes) {
  (void)heads, (void)kv_heads, (void)head_dim, (void)max_nodes;
  return 0;
}

extern "C" int tjk_tree_attention(const void* q, int64_t ld_q_token, int64_t ld_q_head, const tjk_paged_cache* cache,
                                  const int32_t* block_table, int64_t ld_table, int64_t table_cols,
                                  const int32_t* ctx_lens, const int32_t* cu_nodes, const uint64_t* tree_mask, void* out,
                                  int64_t ld_out, int64_t tokens, int batch, int heads, int max_nodes, float scale,
                                  void* workspace, size_t workspace_bytes, int* index_errors, void* stream) {
  const char* const who = "tjk_tree_attention";
  if (const int bad = check_cache(who, cache)) return bad;
  if (tokens < 0 || batch < 0 || heads <= 0 || max_nodes < 0 || table_cols < 0)
    return fail(TJK_EINVAL, "%s: bad shape tokens=%lld batch=%d heads=%d max_nodes=%d", who, (long long)tokens, batch, heads,
                max_nodes);
  if (heads % cache->kv_heads)
    return fail(TJK_EINVAL, "%s: %d heads are no multiple of %d key heads", who, heads, cache->kv_heads);
  if (max_nodes > 64) return fail(TJK_EUNSUPPORTED, "%s: max_nodes=%d exceeds 64", who, max_nodes);
  if (tokens > INT32_MAX || table_cols > INT32_MAX || (int64_t)batch * heads * 64 > INT32_MAX)
    return fail(TJK_EUNSUPPORTED, "%s: too large", who);
  if (tokens == 0 || batch == 0 || max_nodes == 0) return TJK_OK;
  if (!q || !out || !ctx_lens || !cu_nodes || (table_cols > 0 && !block_table))
    return fail(TJK_EINVAL, "%s: null pointer", who);
  if (ld_table < table_cols || ld_out < (int64_t)heads * cache->head_dim || ld_q_head < cache->head_dim || ld_q_token < 0)
    return fail(TJK_EINVAL, "%s: leading dimension too small", who);
  if (ld_q_token % 8 || ld_q_head % 8 || ld_out % 8)
    return fail(TJK_EUNSUPPORTED, "%s: strides must be multiples of 8", who);
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15 || (uintptr_t)tree_mask & 7)
    return fail(TJK_EUNSUPPORTED, "%s: misaligned pointer", who);
  if (workspace_bytes < tjk_tree_attention_bytes(heads, cache->kv_heads, cache->head_dim, max_nodes))
    return fail(TJK_EINVAL, "%s: workspace too small", who);
  const TreeArgs a{static_cast<const char*>(q), 2 * ld_q_token, 2 * ld_q_head, paged(*cache), block_table, ld_table,
                   (int)table_cols, ctx_lens, cu_nodes, tree_mask, static_cast<char*>(out), 2 * ld_out, scale, index_errors,
                   tokens, batch, heads, heads / cache->kv_heads, cache->head_dim / 8, max_nodes};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const unsigned grid = (unsigned)(batch * heads * max_nodes);
  if (cache->dtype == TJK_F16) tree_simple_kernel<f16><<<grid, 256, 0, s>>>(a);
  else tree_simple_kernel<bf16><<<grid, 256, 0, s>>>(a);
  return check_launch(who);
}

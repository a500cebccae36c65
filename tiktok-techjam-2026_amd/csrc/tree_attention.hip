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
  float scale;  // with log2(e): scores are exponents of 2
  float* parts;  // workspace: two partial results per workgroup
  int* index_errors;
  int64_t tokens;
  int batch, kv_heads, group, hd8, max_nodes;
};

// ---------------------------------------------------------------- work
//
// An item is a block of rows of one (sequence, key head): rows m = node * group +
// query head, ROWS of them.  Its keys are cut into tiles of 32, all items' tiles
// are numbered through, and every workgroup takes an equal stretch of them:
// lengths are known on the device only, and a long sequence next to short ones
// is split as finely as it needs.  A stretch that is a whole item writes its rows;
// else it leaves the rows' sums, with their exponent offset, in the workspace, and
// a second launch joins them.

constexpr int kTile = 32;     // keys of a tile
constexpr int kMinTiles = 8;  // least tiles of a workgroup: below, the joining costs more than the splitting gives

struct Seq {
  int b, n, mbs;       // sequence, its nodes, its row blocks
  int64_t first;       // its first row
  int64_t ctx, end;    // tokens behind it, positions that it sees
  int64_t tiles;       // of an item
  int64_t before;      // tiles before it
};

// A lane's sequence b (< batch): everything but `before`.
__device__ __forceinline__ Seq lane_seq(const TreeArgs& a, int b, int rows) {
  Seq q{};
  q.b = b;
  if (b < a.batch) {
    const int lo = max(a.cu_nodes[b], 0), hi = a.cu_nodes[b + 1];
    q.first = lo;
    q.n = (int)min((int64_t)min(max((int64_t)hi - lo, (int64_t)0), (int64_t)a.max_nodes), max(a.tokens - lo, (int64_t)0));
    q.ctx = max(a.ctx_lens[b], 0);
    q.end = min(q.ctx + q.n, (int64_t)a.table_cols << a.cache.shift);
    q.tiles = q.n > 0 ? max((q.end + kTile - 1) / kTile, (int64_t)1) : 0;
    q.mbs = (q.n * a.group + rows - 1) / rows;
  }
  return q;
}

__device__ __forceinline__ int64_t lane_i64(int64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane), hi = __builtin_amdgcn_readlane((int)(v >> 32), lane);
  return (int64_t)((uint64_t)hi << 32 | lo);
}

__device__ __forceinline__ int64_t wave_sum_i64(int64_t v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return lane_i64(v, 0);
}

// Tiles of the whole batch.
__device__ __forceinline__ int64_t all_tiles(const TreeArgs& a, int rows) {
  int64_t sum = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const Seq q = lane_seq(a, b0 + (int)(threadIdx.x & 63), rows);
    sum += q.tiles * q.mbs * a.kv_heads;
  }
  return wave_sum_i64(sum);
}

// The sequence that tile `at` (< all_tiles) belongs to, the same in every lane.
__device__ __forceinline__ Seq find_seq(const TreeArgs& a, int rows, int64_t at) {
  const int lane = threadIdx.x & 63;
  int64_t base = 0;
  for (int b0 = 0;; b0 += 64) {
    const Seq q = lane_seq(a, b0 + lane, rows);
    int64_t incl = q.tiles * q.mbs * a.kv_heads;
    const int64_t mine = incl;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t up = __shfl_up(incl, d);
      incl += lane >= d ? up : 0;
    }
    const uint64_t past = __ballot(base + incl > at);
    if (past != 0 || b0 + 64 >= a.batch) {
      const int l = past ? __ffsll((unsigned long long)past) - 1 : 0;
      Seq r;
      r.b = b0 + l;
      r.n = __builtin_amdgcn_readlane(q.n, l);
      r.mbs = __builtin_amdgcn_readlane(q.mbs, l);
      r.first = lane_i64(q.first, l);
      r.ctx = lane_i64(q.ctx, l);
      r.end = lane_i64(q.end, l);
      r.tiles = lane_i64(q.tiles, l);
      r.before = base + lane_i64(incl - mine, l);
      return r;
    }
    base += lane_i64(incl, 63);
  }
}

// Workgroup w of n takes tiles [share(w), share(w + 1)).
struct Split {
  int64_t total;
  int n;
  __device__ __forceinline__ Split(int64_t tiles, int most)
      : total(tiles), n((int)min((int64_t)most, max((tiles + kMinTiles - 1) / kMinTiles, (int64_t)1))) {}
  __device__ __forceinline__ int64_t share(int w) const { return total * w / n; }
  // the workgroup whose stretch holds tile x
  __device__ __forceinline__ int holder(int64_t x) const {
    int w = (int)((x * n + n - 1) / total);  // the last w with share(w) <= x, or one beside it
    while (w > 0 && (w >= n || share(w) > x)) --w;
    while (w + 1 < n && share(w + 1) <= x) ++w;
    return w;
  }
};

// ----------------------------------------------------------- one stretch
//
// Both products are computed transposed, S^T = K Q^T and O^T += V^T P^T, with
// 16 x 16 x 32 MFMAs: a lane holds one row's scores, so the softmax needs other
// lanes only when a row's offset moves.  Fragments: lane l has row or column
// l % 16 and elements 8 (l / 16) .. + 7 of the contraction; results: column l % 16,
// rows 4 (l / 16) .. + 3.  So the scores of two blocks of 16 keys are, as they lie,
// the fragment of the product with V if its contraction index 8 g + j stands for
// key 16 (j / 4) + 4 g + j % 4, which is what two transposing LDS reads of V give.
//
// Tiles are copied from their pages into LDS by DMA, 16-byte pieces swizzled:
// piece c of row r at c ^ swz(r).  Rows past the end and pieces past head_dim lie
// outside the descriptor's range and arrive as zeros.
//
// RW = 1 (up to 64 rows): the four waves take tiles in turn, each with NST slots of its
// own, and meet only to join their sums: no barrier in the loop.  Copies run ahead
// by NST tiles, K and V apart.  RW = 4 (more rows): the waves have 16 NB rows each
// and share the tiles, in a ring of NST, one barrier a tile.

constexpr uint32_t kPast = 0x80000000u;  // beyond any descriptor's range
constexpr float kLazy = 8.0f;            // a row's offset follows its scores when they pass it by 2^8

template <typename T> struct Mfma16;
template <> struct Mfma16<bf16> {
  static __device__ __forceinline__ f32x4 mma(const bf16x8& a, const bf16x8& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mfma16<f16> {
  static __device__ __forceinline__ f32x4 mma(const f16x8& a, const f16x8& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// Over the lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float column_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float column_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

__device__ __forceinline__ u32x4 range_of(const char* p, uint32_t bytes) {
  const uint64_t x = (uint64_t)(uintptr_t)p;
  return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)x),
               (uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) & 0xffffu,
               (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}

template <int HD, int NB, int RW, int NST>
struct TreeShape {
  static constexpr int ROWS = 16 * NB * RW;
  static constexpr int RB = 2 * HD;             // bytes of a row in LDS
  static constexpr int TB = kTile * RB;         // of a tile's keys or values
  static constexpr int RING = (RW == 1 ? 4 : 1) * NST * 2 * TB;
  static constexpr int JOIN = RW == 1 ? 2 * (NB * HD * 64 + NB * 512) : 0;  // two waves' sums
  static constexpr int LDS = RING > JOIN ? RING : JOIN;
  static constexpr int PART = ROWS * (HD + 2);  // floats of a partial result
};

template <typename T, int HD, int NB, int RW, int NST, int OCC>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(OCC, OCC))) void tree_attention_kernel(TreeArgs a) {
  typedef TreeShape<HD, NB, RW, NST> Sh;
  typedef typename Mfma<T>::frag Frag;
  constexpr int RB = Sh::RB, TB = Sh::TB, CPR = RB / 16, RPI = 64 / CPR;
  constexpr int KC = HD / 32, HT = HD / 16;
  constexpr int NK = TB / 1024;         // DMA instructions of a tile's keys
  constexpr int NV = 16 / RPI;          // of 16 rows
  __shared__ __attribute__((aligned(1024))) char smem[Sh::LDS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;

  const int64_t total = all_tiles(a, Sh::ROWS);
  if (total == 0) return;
  const Split split(total, gridDim.x);
  // neighbouring stretches on one XCD
  const int per = gridDim.x / 8;
  const int w = (int)(blockIdx.x % 8) * per + blockIdx.x / 8;
  if (w >= split.n) return;
  const int64_t stop = split.share(w + 1);
  int64_t at = split.share(w);
  if (at >= stop) return;

  const uint32_t lds = (uint32_t)(uintptr_t)(lds_void*)smem;
  auto swz = [](int r) {
    return CPR == 16 ? ((r >> 3 & 1) | (r & 7) << 1) : ((r >> 3 & 1) | (r & 6));
  };
  uint32_t voff[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int r = i * RPI + lane / CPR, c = (lane % CPR) ^ swz(r);
    voff[i] = (uint32_t)r * a.cache.row_bytes + (c < a.hd8 ? 16u * c : kPast);
  }
  // fragment addresses within a tile
  int kaddr[KC];
#pragma unroll
  for (int c = 0; c < KC; ++c) kaddr[c] = col * RB + (((4 * c + g) ^ swz(col)) << 4);
  const int vrow = 4 * g + (col >> 2);
  int vaddr[HT];
#pragma unroll
  for (int h = 0; h < HT; ++h) vaddr[h] = vrow * RB + (((2 * h + (lane >> 1 & 1)) ^ swz(vrow)) << 4) + 8 * (lane & 1);

  Seq q = find_seq(a, Sh::ROWS, at);
  int slot = 1;  // of this workgroup's next partial result
  while (at < stop) {
    if (at >= q.before + q.tiles * q.mbs * a.kv_heads) q = find_seq(a, Sh::ROWS, at);
    const int64_t off = at - q.before;
    const int item = (int)(off / q.tiles);
    const int64_t t0 = off - item * q.tiles, t1 = min(q.tiles, t0 + (stop - at));
    at += t1 - t0;
    const int kh = item / q.mbs, mb = item - kh * q.mbs;
    const int rows = q.n * a.group, m0 = mb * Sh::ROWS + (RW == 1 ? 0 : wave * 16 * NB);
    const int64_t end = q.end;
    const char* const kbase = a.cache.k + kh * a.cache.head_bytes;
    const char* const vbase = a.cache.v + kh * a.cache.head_bytes;
    const int32_t* const table = a.table + q.b * a.ld_table;

    // ---- this lane's rows: queries, visible nodes
    Frag qf[NB][KC];
    uint64_t bits[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int m = m0 + 16 * i + col;
      const bool live = m < rows;
      const int node = live ? m / a.group : 0, head = kh * a.group + (live ? m - node * a.group : 0);
      const int64_t t = q.first + node;
      const T* const src = reinterpret_cast<const T*>(a.q + t * a.q_token_bytes + head * a.q_head_bytes);
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const bool in = live && 4 * c + g < a.hd8;
        Frag f = Mfma<T>::load(src + (4 * c + g < a.hd8 ? 8 * (4 * c + g) : 0));
        const u32x4 zero = {0, 0, 0, 0};
        qf[i][c] = in ? f : __builtin_bit_cast(Frag, zero);
      }
      bits[i] = a.mask ? a.mask[t] : ~0ull >> (63 - node);
    }

    // ---- pages of the next 64 tiles: lane j has those of tile first + j * STEP,
    // the first and the second 16 positions'
    constexpr int STEP = RW == 1 ? 4 : 1;
    const int64_t mine = RW == 1 ? t0 + wave : t0;
    const int count = mine < t1 ? (int)((t1 - mine + STEP - 1) / STEP) : 0;
    int page[2];
    auto load_pages = [&](int i0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t x = (mine + (int64_t)(i0 + lane) * STEP) * kTile + 16 * h;
        const bool in = i0 + lane < count && x < end;
        page[h] = page_of(table, in ? (int)(x >> a.cache.shift) : 0, a.cache.pages);
        if (in && page[h] < 0 && kh == 0 && mb == 0 && (RW == 1 || wave == 0) && a.index_errors) atomicAdd(a.index_errors, 1);
        if (!in) page[h] = -1;
      }
    };
    if (kh == 0 && mb == 0 && t0 == 0 && threadIdx.x == 0 && a.index_errors && end < q.ctx + q.n) atomicAdd(a.index_errors, 1);
    page[0] = page[1] = -1;
    if (end > 0) load_pages(0);
    // 16 rows of keys or values: descriptor of tile i's half h
    auto half_range = [&](const char* base, int i, int h) {
      const int pg = __builtin_amdgcn_readlane(page[h], i & 63);
      const int64_t x = (mine + (int64_t)i * STEP) * kTile + 16 * h;
      const int left = (int)min(max(end - x, (int64_t)0), (int64_t)16);
      const char* const p = base + (int64_t)max(pg, 0) * a.cache.page_bytes +
                            (int64_t)((int)x & ((1 << a.cache.shift) - 1)) * a.cache.row_bytes;
      return range_of(p, pg < 0 || i >= count ? 0 : (uint32_t)left * a.cache.row_bytes);
    };
    // halves of tile i without a page: bits 0 and 1
    auto pageless = [&](int i) {
      return (__builtin_amdgcn_readlane(page[0], i & 63) < 0 ? 1 : 0) | (__builtin_amdgcn_readlane(page[1], i & 63) < 0 ? 2 : 0);
    };
    // tile i's keys (or values) to LDS byte `to`
    auto copy = [&](const char* base, int i, uint32_t to) {
      if constexpr (RW == 1) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x4 r = half_range(base, i, h);
#pragma unroll
          for (int u = 0; u < NV; ++u) lds_dma16(r, voff[u], to + (h * NV + u) * 1024);
        }
      } else {
#pragma unroll
        for (int u = 0; u < (NK + 3) / 4; ++u) {
          const int k = wave + 4 * u;
          const u32x4 r = half_range(base, i, k / NV);
          uint32_t v = voff[0];
#pragma unroll
          for (int j = 1; j < NV; ++j) v = k % NV == j ? voff[j] : v;
          lds_dma16(r, v, to + k * 1024);
        }
      }
    };

    f32x4 o[NB][HT];
    float m_off[NB], l[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      m_off[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int h = 0; h < HT; ++h) o[i][h] = f32x4{0, 0, 0, 0};
    }

    // ---- the products of tile i, its keys and values in LDS at kt and vt
    auto scores = [&](const char* kt, f32x4 (&s)[NB][2]) {
      Frag kf[2][KC];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int c = 0; c < KC; ++c) kf[b][c] = *reinterpret_cast<const Frag*>(kt + 16 * b * RB + kaddr[c]);
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          s[i][b] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < KC; ++c) s[i][b] = Mfma16<T>::mma(kf[b][c], qf[i][c], s[i][b]);
        }
    };
    // whether this lane's row i sees key x + k (k: of the tile)
    auto sees = [&](int i, int64_t x, int k, int none) {
      const int64_t p = x + k;
      const bool tree = p < q.ctx || (p - q.ctx < 64 && (bits[i] >> ((p - q.ctx) & 63) & 1));
      return p < end && tree && !(none >> (k >> 4) & 1);
    };
    auto softmax = [&](f32x4 (&s)[NB][2], Frag (&p)[NB], int64_t x, bool masked, int none) {
      bool moves = false;
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        float top = -INFINITY;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float v = s[i][b][r] * a.scale;
            if (masked) v = sees(i, x, 16 * b + 4 * g + r, none) ? v : -INFINITY;
            s[i][b][r] = v;
            top = fmaxf(top, v);
          }
        moves |= top > m_off[i] + kLazy;
      }
      if (__any(moves)) {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          float top = -INFINITY;
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) top = fmaxf(top, s[i][b][r]);
          const float m = fmaxf(m_off[i], column_max(top));
          const float keep = m_off[i] == m ? 1.f : __builtin_amdgcn_exp2f(m_off[i] - m);
          m_off[i] = m;
          l[i] *= keep;
#pragma unroll
          for (int h = 0; h < HT; ++h) o[i][h] *= keep;
        }
      }
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const float base = m_off[i] == -INFINITY ? 0.f : m_off[i];
        float e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = __builtin_amdgcn_exp2f(s[i][j >> 2][j & 3] - base);
        p[i] = Mfma<T>::pack(e);
        // sums of the rounded weights, those that the product uses
        l[i] = Mfma<T>::sum8(p[i], l[i]);
      }
    };
    // Infinities and NaN among a tile's values: a weight of zero would not keep them
    // from a row that does not see them.  They are added to the rows that do, and
    // the product finds zeros in their place.  (Tiles of the c tokens need none of
    // this: every row sees those.)
    auto bad_values = [&](const char* vt) -> uint32_t {
      const int row = lane >> 1;
      bool bad = false;
#pragma unroll
      for (int c = 0; c < CPR / 2; ++c) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(vt + row * RB + ((lane & 1) * (CPR / 2) + c) * 16);
        constexpr uint32_t E = std::is_same<T, bf16>::value ? 0x7f80u : 0x7c00u;
#pragma unroll
        for (int k = 0; k < 4; ++k) bad |= (v[k] & E) == E || (v[k] >> 16 & E) == E;
      }
      const uint64_t m = __ballot(bad);
      uint32_t keys = 0;  // bits 2 k, 2 k + 1 -> k; rare
      for (uint64_t x = m; x; x &= x - 1) keys |= 1u << ((__ffsll((unsigned long long)x) - 1) >> 1);
      return keys;
    };
    auto add_bad = [&](const char* vt, uint32_t keys, int64_t x, int none) {
      for (; keys; keys &= keys - 1) {
        const int k = __ffs(keys) - 1;
        const int sw = swz(k & 15);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const bool seen = sees(i, x, k, none);
#pragma unroll
          for (int h = 0; h < HT; ++h) {
            const int c = 2 * h + (g >> 1);
            const uint2 raw = *reinterpret_cast<const uint2*>(vt + k * RB + ((c ^ sw) << 4) + 8 * (g & 1));
            const float4 v = Quad<T>::to(raw);
            const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (seen && !(fabsf(e[r]) < INFINITY)) o[i][h][r] += e[r];
          }
        }
      }
    };
    auto clear_bad = [&](char* vt) {
      const int row = lane >> 1;
      for (int c = 0; c < CPR / 2; ++c) {
        u32x4* const at = reinterpret_cast<u32x4*>(vt + row * RB + ((lane & 1) * (CPR / 2) + c) * 16);
        u32x4 v = *at;
        constexpr uint32_t E = std::is_same<T, bf16>::value ? 0x7f80u : 0x7c00u;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if ((v[k] & E) == E) v[k] &= 0xffff0000u;
          if ((v[k] >> 16 & E) == E) v[k] &= 0xffffu;
        }
        *at = v;
      }
    };
    auto products = [&](const char* vt, const Frag (&p)[NB]) {
#pragma unroll
      for (int h = 0; h < HT; ++h) {
        typedef short v4s __attribute__((ext_vector_type(4)));
        typedef short v8s __attribute__((ext_vector_type(8)));
        const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(vt + vaddr[h]));
        const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(vt + vaddr[h] + 16 * RB));
        const v8s both = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        const Frag vf = __builtin_bit_cast(Frag, both);
#pragma unroll
        for (int i = 0; i < NB; ++i) o[i][h] = Mfma16<T>::mma(vf, p[i], o[i][h]);
      }
    };

    if constexpr (RW == 1) {
      const uint32_t ring = lds + wave * (NST * 2 * TB);
      char* const mem = smem + wave * (NST * 2 * TB);
      int lost[NST];  // of the tiles in the slots
#pragma unroll
      for (int s = 0; s < NST; ++s) {
        copy(kbase, s, ring + s * 2 * TB);
        copy(vbase, s, ring + s * 2 * TB + TB);
        lost[s] = pageless(s);
      }
      for (int i0 = 0; i0 < count; i0 += NST) {
#pragma unroll
        for (int s = 0; s < NST; ++s) {
          const int i = i0 + s;
          if (NST > 1 && i >= count) break;
          char* const kt = mem + s * 2 * TB;
          char* const vt = kt + TB;
          const int64_t x = (mine + (int64_t)i * STEP) * kTile;
          const int none = lost[s];
          const bool masked = x + kTile > q.ctx || none != 0;
          if (((i + NST) & 63) == 0 && i + NST < count) load_pages(i + NST);
          f32x4 sc[NB][2];
          Frag p[NB];
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NK * (2 * NST - 1)) : "memory");
          scores(kt, sc);
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          copy(kbase, i + NST, ring + s * 2 * TB);
          lost[s] = pageless(i + NST);
          softmax(sc, p, x, masked, none);
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NK * (2 * NST - 1)) : "memory");
          if (masked) {
            const uint32_t keys = bad_values(vt);
            if (keys) {
              add_bad(vt, keys, x, none);
              clear_bad(vt);
              asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            }
          }
          products(vt, p);
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          copy(vbase, i + NST, ring + s * 2 * TB + TB);
        }
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      // ---- join the four waves' sums: 2 and 3 into 0 and 1, then 1 into 0
      __syncthreads();
#pragma unroll
      for (int half = 2; half >= 1; half >>= 1) {
        float4* const xo = reinterpret_cast<float4*>(smem + (wave & (half - 1)) * (NB * HD * 64 + NB * 512));
        float* const xm = reinterpret_cast<float*>(xo + NB * HT * 64);
        if (wave >= half && wave < 2 * half) {
#pragma unroll
          for (int i = 0; i < NB; ++i) {
#pragma unroll
            for (int h = 0; h < HT; ++h) xo[(i * HT + h) * 64 + lane] = make_float4(o[i][h][0], o[i][h][1], o[i][h][2], o[i][h][3]);
            xm[i * 128 + lane] = m_off[i];
            xm[i * 128 + 64 + lane] = l[i];
          }
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            const float m2 = xm[i * 128 + lane], m = fmaxf(m_off[i], m2);
            const float f1 = m_off[i] == m ? 1.f : __builtin_amdgcn_exp2f(m_off[i] - m);
            const float f2 = m2 == m ? 1.f : __builtin_amdgcn_exp2f(m2 - m);
            m_off[i] = m;
            l[i] = l[i] * f1 + xm[i * 128 + 64 + lane] * f2;
#pragma unroll
            for (int h = 0; h < HT; ++h) {
              const float4 v = xo[(i * HT + h) * 64 + lane];
              o[i][h][0] = o[i][h][0] * f1 + v.x * f2;
              o[i][h][1] = o[i][h][1] * f1 + v.y * f2;
              o[i][h][2] = o[i][h][2] * f1 + v.z * f2;
              o[i][h][3] = o[i][h][3] * f1 + v.w * f2;
            }
          }
        }
        __syncthreads();
      }
    } else {
      constexpr int NI = 2 * ((NK + 3) / 4);  // a wave's DMA instructions of a tile
      int lost[NST];  // of tile i and those behind it
#pragma unroll
      for (int s = 0; s < NST - 1; ++s) {
        copy(kbase, s, lds + s * 2 * TB);
        copy(vbase, s, lds + s * 2 * TB + TB);
        lost[s] = pageless(s);
      }
      int s = 0;
      for (int i = 0; i < count; ++i) {
        const int64_t x = (mine + i) * kTile;
        const int none = lost[0];
        const bool masked = x + kTile > q.ctx || none != 0;
        if (((i + NST - 1) & 63) == 0 && i + NST - 1 < count) load_pages(i + NST - 1);
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(NI * (NST - 2)) : "memory");
        const int next = s == 0 ? NST - 1 : s - 1;
        copy(kbase, i + NST - 1, lds + next * 2 * TB);
        copy(vbase, i + NST - 1, lds + next * 2 * TB + TB);
        lost[NST - 1] = pageless(i + NST - 1);
#pragma unroll
        for (int j = 0; j < NST - 1; ++j) lost[j] = lost[j + 1];
        char* const kt = smem + s * 2 * TB;
        char* const vt = kt + TB;
        f32x4 sc[NB][2];
        Frag p[NB];
        scores(kt, sc);
        softmax(sc, p, x, masked, none);
        if (masked) {
          const uint32_t keys = bad_values(vt);  // the same in every wave
          if (keys) {
            add_bad(vt, keys, x, none);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (wave == 0) clear_bad(vt);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
          }
        }
        products(vt, p);
        s = s == NST - 1 ? 0 : s + 1;
      }
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }

    // ---- the rows, or what the joining launch needs of them
    const bool whole = t0 == 0 && t1 == q.tiles;
    if (RW == 1 && wave != 0) continue;
    const int64_t part = 2 * (int64_t)w + (t0 == 0 ? 1 : 0);
    (void)slot;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int m = m0 + 16 * i + col;
      const float sum = column_sum(l[i]);
      if (m >= rows) continue;
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
        const int node = m / a.group, head = kh * a.group + m - node * a.group;
        T* const dst = reinterpret_cast<T*>(a.out + (q.first + node) * a.out_bytes) + (int64_t)head * (8 * a.hd8);
#pragma unroll
        for (int h = 0; h < HT; ++h)
          if (16 * h < 8 * a.hd8)
            *reinterpret_cast<typename Quad<T>::raw*>(dst + 16 * h + 4 * g) =
                Quad<T>::from(make_float4(o[i][h][0] * inv, o[i][h][1] * inv, o[i][h][2] * inv, o[i][h][3] * inv));
      } else {
        float* const dst = a.parts + part * Sh::PART + (int64_t)(m - mb * Sh::ROWS) * HD;
#pragma unroll
        for (int h = 0; h < HT; ++h)
          *reinterpret_cast<float4*>(dst + 16 * h + 4 * g) = make_float4(o[i][h][0], o[i][h][1], o[i][h][2], o[i][h][3]);
        float* const ml = a.parts + part * Sh::PART + Sh::ROWS * HD + 2 * (m - mb * Sh::ROWS);
        if (g == 0) *reinterpret_cast<float2*>(ml) = make_float2(m_off[i], sum);
      }
    }
  }
}

// Joins the stretches of an item: a workgroup takes kJoinRows rows of it, 16
// lanes a row (eight or four columns each), the stretches in turn over its
// row groups.  The order is that of the keys, whoever finished first.
constexpr int kJoinRows = 16;

template <typename T, int HD, int ROWS>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a, int most) {
  constexpr int V = HD / 16, PART = ROWS * (HD + 2);
  const int64_t total = all_tiles(a, ROWS);
  if (total == 0) return;
  const Split split(total, most);
  const int blocks = (ROWS + kJoinRows - 1) / kJoinRows;
  const int mbs = (a.max_nodes * a.group + ROWS - 1) / ROWS;
  int rest = blockIdx.x;
  const int rb = rest % blocks;
  rest /= blocks;
  const int mb = rest % mbs;
  rest /= mbs;
  const int kh = rest % a.kv_heads, b = rest / a.kv_heads;
  // this sequence, and the tiles before it
  int64_t before = 0;
  for (int b0 = 0; b0 < b; b0 += 64) {
    const int l = b0 + (int)(threadIdx.x & 63);
    if (l < b) {
      const Seq q = lane_seq(a, l, ROWS);
      before += q.tiles * q.mbs * a.kv_heads;
    }
  }
  before = wave_sum_i64(before);
  const Seq q = lane_seq(a, b, ROWS);
  const int row = rb * kJoinRows + (threadIdx.x >> 4);
  const int m = mb * ROWS + row;
  if (q.n == 0 || mb >= q.mbs) return;
  const int64_t first = before + ((int64_t)kh * q.mbs + mb) * q.tiles, last = first + q.tiles - 1;
  const int w0 = split.holder(first), w1 = split.holder(last);
  if (w0 == w1) return;  // one workgroup had all of it
  if (row >= ROWS || m >= q.n * a.group) return;
  const int c0 = (threadIdx.x & 15) * V;
  float top = -INFINITY, sum = 0.f, o[V];
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = 0.f;
  for (int w = w0; w <= w1; ++w) {
    // the first stretch may begin in the middle of its workgroup's
    const float* const part = a.parts + (2 * (int64_t)w + (w == w0 ? 1 : 0)) * PART;
    const float2 ml = *reinterpret_cast<const float2*>(part + ROWS * HD + 2 * row);
    const float t = fmaxf(top, ml.x);
    const float f1 = top == t ? 1.f : __builtin_amdgcn_exp2f(top - t), f2 = ml.x == t ? 1.f : __builtin_amdgcn_exp2f(ml.x - t);
    top = t;
    sum = sum * f1 + ml.y * f2;
    const float4* const src = reinterpret_cast<const float4*>(part + row * HD + c0);
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 v = src[i / 4];
      o[i] = o[i] * f1 + v.x * f2;
      o[i + 1] = o[i + 1] * f1 + v.y * f2;
      o[i + 2] = o[i + 2] * f1 + v.z * f2;
      o[i + 3] = o[i + 3] * f1 + v.w * f2;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  const int node = m / a.group, head = kh * a.group + m - node * a.group;
  T* const dst = reinterpret_cast<T*>(a.out + (q.first + node) * a.out_bytes) + (int64_t)head * (8 * a.hd8);
  if (c0 < 8 * a.hd8) {
#pragma unroll
    for (int i = 0; i < V; i += 4)
      *reinterpret_cast<typename Quad<T>::raw*>(dst + c0 + i) =
          Quad<T>::from(make_float4(o[i] * inv, o[i + 1] * inv, o[i + 2] * inv, o[i + 3] * inv));
  }
}

// ---------------------------------------------------------------- variants

// Workgroups of a launch: the CUs times those that a CU holds.
constexpr int kCus = 256;

template <int HD_, int NB_, int RW_, int NST_, int OCC_>
struct Variant {
  static constexpr int HD = HD_, NB = NB_, RW = RW_, NST = NST_, OCC = OCC_;
  typedef TreeShape<HD, NB, RW, NST> Sh;
  static constexpr int GRID = kCus * OCC;
  static constexpr size_t BYTES = (size_t)2 * GRID * Sh::PART * sizeof(float);
};

// Calls f with the variant for a head_dim and the rows of the largest tree.
template <typename F>
static auto with_variant(int head_dim, int rows, F&& f) {
  if (head_dim <= 64) {
    if (rows <= 16) return f(Variant<64, 1, 1, 2, 2>{});
    if (rows <= 32) return f(Variant<64, 2, 1, 2, 2>{});
    if (rows <= 64) return f(Variant<64, 4, 1, 2, 2>{});
    if (rows <= 128) return f(Variant<64, 2, 4, 3, 2>{});
    return f(Variant<64, 4, 4, 3, 2>{});
  }
  if (rows <= 16) return f(Variant<128, 1, 1, 1, 2>{});
  if (rows <= 32) return f(Variant<128, 2, 1, 1, 2>{});
  if (rows <= 64) return f(Variant<128, 4, 1, 2, 1>{});
  if (rows <= 128) return f(Variant<128, 2, 4, 3, 2>{});
  return f(Variant<128, 4, 4, 3, 2>{});
}

template <typename T, typename V>
static int launch_tree(const TreeArgs& a, hipStream_t s) {
  constexpr int ROWS = V::Sh::ROWS;
  tree_attention_kernel<T, V::HD, V::NB, V::RW, V::NST, V::OCC><<<V::GRID, 256, 0, s>>>(a);
  if (const int bad = check_launch("tjk_tree_attention")) return bad;
  const int64_t mbs = (a.max_nodes * a.group + ROWS - 1) / ROWS;
  const int64_t grid = (int64_t)a.batch * a.kv_heads * mbs * ((ROWS + kJoinRows - 1) / kJoinRows);
  tree_join_kernel<T, V::HD, ROWS><<<(unsigned)grid, 256, 0, s>>>(a, V::GRID);
  return check_launch("tjk_tree_attention");
}

}  // namespace tjk

using namespace tjk;

extern "C" size_t tjk_tree_attention_bytes(int heads, int kv_heads, int head_dim, int max_nodes) {
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || head_dim <= 0 || head_dim % 16 || head_dim > 128 || max_nodes <= 0 ||
      max_nodes > 64 || heads > 65536)
    return 0;
  return with_variant(head_dim, max_nodes * (heads / kv_heads), [](auto v) { return decltype(v)::BYTES; });
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
  if (heads > 65536 || tokens > INT32_MAX || table_cols > INT32_MAX || (int64_t)batch * heads * 64 > INT32_MAX)
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
  if (!workspace) return fail(TJK_EINVAL, "%s: null workspace", who);
  const size_t need = tjk_tree_attention_bytes(heads, cache->kv_heads, cache->head_dim, max_nodes);
  if (workspace_bytes < need)
    return fail(TJK_EINVAL, "%s: a workspace of %zu bytes, %zu needed", who, workspace_bytes, need);
  const float log2e = 1.44269504088896340736f;
  const TreeArgs a{static_cast<const char*>(q), 2 * ld_q_token, 2 * ld_q_head, paged(*cache), block_table, ld_table,
                   (int)table_cols, ctx_lens, cu_nodes, tree_mask, static_cast<char*>(out), 2 * ld_out, scale * log2e,
                   static_cast<float*>(workspace), index_errors, tokens, batch, cache->kv_heads, heads / cache->kv_heads,
                   cache->head_dim / 8, max_nodes};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return with_variant(cache->head_dim, max_nodes * a.group, [&](auto v) {
    return cache->dtype == TJK_F16 ? launch_tree<f16, decltype(v)>(a, s) : launch_tree<bf16, decltype(v)>(a, s);
  });
}

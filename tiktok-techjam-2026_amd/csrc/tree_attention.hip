// Attention of drafted tokens over the paged cache.
//
// A sequence has c tokens behind it, whose keys and values are positions 0 ..
// c - 1 of its pages, and n <= 64 nodes (drafted tokens, parents first) at
// positions c .. c + n - 1.  A node sees all of the c tokens and the nodes that
// its mask names.  Query head h reads key head h / (heads / kv_heads).

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "paged_cache.h"

namespace tjk {

struct TreeArgs {
  const char* q;
  int64_t q_token_bytes, q_head_bytes;
  Paged cache;
  const int32_t* table;
  int64_t ld_table;
  const int32_t* ctx_lens;
  const int32_t* cu_nodes;
  const uint64_t* mask;
  char* out;
  int64_t out_bytes;  // of a row
  float scale;  // its size, with log2(e): scores are exponents of 2
  int* counters;  // workspace: two per workgroup and level of joining, zero between launches
  float* parts;   // two partial results per workgroup
  int* index_errors;
  uint32_t flip;  // the signs of two queries' elements, if the scale is negative
  int room;       // positions that the block table holds
  int tokens, batch, kv_heads, group, hd8, max_nodes;
  int most_mbs;   // row blocks of the largest tree
  int direct;     // an item is one workgroup's
};

// ---------------------------------------------------------------- work
//
// An item is a block of rows of one (sequence, key head): rows m = node * group +
// query head, ROWS of them.  Its keys are cut into tiles of 32.  An item counts
// COST units, for what it costs beside its tiles, and one for each tile; all
// items' units are numbered through (all first row blocks, then all second ones, and so
// on; in each the sequences, their key heads and tiles), and every workgroup takes an equal stretch of
// them: lengths are known on the device only, and a long sequence next to short
// ones is split as finely as it needs.  A stretch that is a whole item writes its rows;
// else it leaves the rows' sums, with their exponent offset, in the workspace.  Of
// eight neighbouring stretches of an item the workgroup that comes last (a counter
// says which) joins the eight, of eight such eights the last one them, and so on;
// always in the order of the keys.  Nobody waits for another, and the counters are
// left at zero.  (One workgroup joining all 64 stretches of an item took 25 us of 70
// for 2 x 99995 tokens.)

constexpr int kTile = 32;     // keys of a tile
constexpr int kJoin = 8;      // sums that are joined at a time
constexpr int kMinUnits = 8;  // of a workgroup: below, the joining costs more than the splitting gives

// The launch's arguments, loaded again: kept over the tiles' loop, they would take
// its scalar registers, and the loop reload them from lanes of a vector register.
typedef const __attribute__((address_space(4))) TreeArgs ConstArgs;
__device__ __forceinline__ ConstArgs& fresh_args() {
  ConstArgs* p = (ConstArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *p;
}
template <typename T>
__device__ __forceinline__ T* in_memory(T* p) {  // (a pointer out of the arguments is one to device memory)
  return (T*)(__attribute__((address_space(1))) T*)p;
}

struct Seq {
  int b, n, mbs;  // sequence, its nodes, its row blocks
  int mb;         // the row block that is meant
  int first;      // its first row
  int ctx, end;   // tokens behind it, positions that it sees
  int tiles;      // of an item
  int before;     // units before it, in front of those of its row block mb
};

// Sequence b (< batch, else nothing): everything but `before`.
template <typename A>
__device__ __forceinline__ Seq load_seq(const A& a, int b, int rows) {
  Seq q{};
  q.b = b;
  if (b < a.batch) {
    const int lo = max(in_memory(a.cu_nodes)[b], 0), hi = max(in_memory(a.cu_nodes)[b + 1], 0);
    q.first = lo;
    q.n = min(min(max(hi - lo, 0), a.max_nodes), max(a.tokens - lo, 0));
    q.ctx = min(max(in_memory(a.ctx_lens)[b], 0), INT32_MAX - 128);
    q.end = min(q.ctx + q.n, a.room);
    q.tiles = q.n > 0 ? max((q.end + kTile - 1) / kTile, 1) : 0;
    q.mbs = (q.n * a.group + rows - 1) / rows;
  }
  return q;
}
// Units of one of its row blocks.
template <typename A>
__device__ __forceinline__ int seq_units(const A& a, const Seq& q, int cost) { return (q.tiles + cost) * a.kv_heads; }

// Inclusive sum over the lanes.
__device__ __forceinline__ int wave_scan(int v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(v, d);
    v += lane >= d ? up : 0;
  }
  return v;
}

// The sequences of a batch, 64 at a time, and the units before and of them: first
// those of all sequences' first row blocks, then of the second ones, and so on.
template <typename Sh>
struct Plan {
  Seq q;  // lane l: sequence first + l
  int first, incl, base, mb;
  template <typename A>
  __device__ __forceinline__ int units(const A& a) const { return q.mbs > mb ? seq_units(a, q, Sh::COST) : 0; }
  template <typename A>
  __device__ __forceinline__ void load(const A& a, int b0) {
    first = b0;
    q = load_seq(a, b0 + (int)(threadIdx.x & 63), Sh::ROWS);
    incl = wave_scan(units(a));
  }
  // all of the batch's units; the first 64 sequences are left loaded
  template <typename A>
  __device__ __forceinline__ int total(const A& a) {
    int sum = 0;
    mb = 0;
    for (int b0 = (a.batch - 1) / 64 * 64; b0 >= 0; b0 -= 64) {
      load(a, b0);
      sum += __builtin_amdgcn_readlane(Sh::MANY ? wave_scan(seq_units(a, q, Sh::COST) * q.mbs) : incl, 63);
    }
    base = 0;
    return sum;
  }
  // The sequence and row block that unit `at` (< total, not before the last one asked
  // for) belongs to, the same in every lane.
  template <typename A>
  __device__ __forceinline__ Seq find(const A& a, int at) {
    while (true) {
      const uint64_t past = __ballot(base + incl > at);
      const bool end = first + 64 >= a.batch;
      if (past != 0 || (end && (!Sh::MANY || mb + 1 >= a.most_mbs))) {
        const int l = past ? __ffsll((unsigned long long)past) - 1 : 0;
        return {first + l, __builtin_amdgcn_readlane(q.n, l), __builtin_amdgcn_readlane(q.mbs, l), mb,
                __builtin_amdgcn_readlane(q.first, l), __builtin_amdgcn_readlane(q.ctx, l),
                __builtin_amdgcn_readlane(q.end, l), __builtin_amdgcn_readlane(q.tiles, l),
                base + __builtin_amdgcn_readlane(incl - units(a), l)};
      }
      base += __builtin_amdgcn_readlane(incl, 63);
      mb += end;
      if (end && first == 0) incl = wave_scan(units(a));
      else load(a, end ? 0 : first + 64);
    }
  }
};

// Of `total` units workgroup w < n takes [share(w), share(w + 1)).
struct Split {
  int n, each, more;  // `more` workgroups take each + 1
  Split() = default;
  __device__ __forceinline__ Split(int total, int most) {
    n = min(most, max((total + kMinUnits - 1) / kMinUnits, 1));
    each = (int)((uint32_t)total / (uint32_t)n);
    more = total - each * n;
  }
  __device__ __forceinline__ int share(int w) const { return w * each + min(w, more); }
  __device__ __forceinline__ int holder(int x) const {  // of unit x
    const int big = more * (each + 1);
    return x < big ? (int)((uint32_t)x / (uint32_t)(each + 1)) : more + (int)((uint32_t)(x - big) / (uint32_t)max(each, 1));
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
// by NST tiles, K and V apart.  RW = 0: the same, but each wave has an item of its own, and
// they do not meet at all (many items of few tiles).  RW = 4 (more rows): the waves have 16 NB rows each
// and share the tiles, in a ring of NST stages of SUB, one barrier a stage.
//
// Weights go to the product with V in the cache's type, as in flash_pipe_kernel: off by
// 2^-8 (bf16) at most each, 2.2e-3 of the result (2-norm) where its own rounding
// is 1.7e-3 (fp16 2.5e-4 and 2.1e-4); a product in two parts would double it.  Everything summed is fp32, the
// sum of the weights that of the rounded ones.
//
// Few rows are bound by memory: 64 single tokens over 512 to 4096, 16 heads of 128
// bf16, 213 us, 5.6 TB/s (a copy of 1 GB reaches 5.1); 2 x 99995 tokens, 4 key heads of
// 64, 57 us (48 on the same ones again), of which the joining takes 12.  8 single tokens
// over up to 512: 8.8 us, launch and passages of memory one after the other (places 2,
// first tiles 1.5, the rest of them 3, joining of the waves 1).  Many rows are bound
// by the matrix and the vector unit and by power: 32 trees of 64 nodes over 1000 to 8192,
// 8 heads of 128 to a key head, 200 to 210 us, 740 to 780 TFLOP/s, and 212 to 262 in the
// first milliseconds after a pause, until the clock has settled (64 over 4000: 313 us,
// 870); matrix unit 32% of the time, vector unit 41%, LDS 18%.  (Before row blocks lay side by side,
// 336 us for the latter: 280 if every page lay in L2, and 280 if keys and values were
// zeros, at the same traffic.)  Per wave 48 rows take 5 to 10% longer than 32, 64
// (one wave a SIMD; two do not fit) 15%, three waves a SIMD do not fit; the next tile's
// scores ahead of the softmax, with a barrier a tile for it, 8 to 15% longer;
// fragments loaded further ahead and wave priorities, no difference.

constexpr uint32_t kPast = 0x80000000u;  // beyond any descriptor's range
// Cache policies: stores through to memory, loads from it, past an XCD's own L2.
constexpr int kThrough = 17, kCoherent = 16;
// A row's offset follows its scores when they pass it by 2^8: most tiles rescale
// nothing, and a weight of up to 256 is no harm in either type.
constexpr float kLazy = 8.0f;
// Weights are 2^kLift above what the offset makes of them (it cancels in the result,
// and all parts of an item share it).  fp16 weights are whole multiples of 2^-24, and
// with the largest at 1 a row of one large weight and 99995 of 2^-25 and less lost them
// all; of 2^7 to 2^15 the largest, the rounding is 2^-32 of it.
template <typename T>
constexpr float kLift = std::is_same<T, f16>::value ? 7.0f : 0.0f;

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

// One LDS DMA (see lds_dma16) with wait states of its own: the compiler does not look
// into inline asm.  Five lie between a VALU write of an SGPR (v_readlane, v_readfirstlane: the
// descriptors are made of such) and a vector memory instruction that reads it, one
// between a write of m0 and a copy into LDS.
__device__ __forceinline__ void copy16(u32x4 rsrc, uint32_t voff, uint32_t lds_addr) {
  asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "{m0}"(lds_addr));
}

// SUB: tiles of a stage of the shared ring (RW = 4).
template <int HD, int NB, int RW, int NST, int SUB>
struct TreeShape {
  static constexpr int ROWS = 16 * NB * (RW > 1 ? RW : 1);
  static constexpr bool MANY = RW > 1;  // trees of more than one row block
  // Units of an item beside its tiles': 9 single tokens over 29 to 4921, 8 heads of 80,
  // 56 us with 0, 30 with 2, 25.6 with 4, 23.9 with 8; 16 trees of 64 nodes, 2 heads of
  // 128 to a key head, 96 with 8, 79 with 16.
  static constexpr int COST = RW <= 1 ? 8 : 16;
  static constexpr int RB = 2 * HD;             // bytes of a row in LDS
  static constexpr int TB = kTile * RB;         // of a tile's keys or values
  static constexpr int RING = (RW <= 1 ? 4 : SUB) * NST * 2 * TB;
  static constexpr int JOIN = RW == 1 ? 2 * (NB * HD * 64 + NB * 512) : 0;  // two waves' sums
  static constexpr int LDS = RING > JOIN ? RING : JOIN;
  static constexpr int PART = ROWS * (HD + 2);  // floats of a partial result
};

template <typename T, int HD, int NB, int RW, int NST, int OCC, int SUB>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(OCC, OCC))) void tree_attention_kernel(TreeArgs args) {
  ConstArgs& a = fresh_args();
  typedef TreeShape<HD, NB, RW, NST, SUB> Sh;
  typedef typename Mfma<T>::frag Frag;
  constexpr int RB = Sh::RB, TB = Sh::TB, CPR = RB / 16, RPI = 64 / CPR;
  constexpr int KC = HD / 32, HT = HD / 16;
  constexpr int NK = TB / 1024;         // DMA instructions of a tile's keys
  constexpr int NV = 16 / RPI;          // of 16 rows
  __shared__ __attribute__((aligned(1024))) char smem[Sh::LDS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;

  // this workgroup's stretch [at, stop) of all units
  Seq q;
  int first64 = 0, base64 = 0;  // the 64 sequences that hold q, the units before them
  Split split{};
  int at, stop, w;
  // Workgroups of one XCD have neighbouring stretches, so that the row blocks of a key
  // head, which read the same keys and values, read them at the same time from its
  // cache: 32 trees of 64 nodes over 1000 to 8192, 8 heads of 128 to a key head, 227 us with
  // row blocks one after the other, 216 and a third of the reads from memory so; 64 trees
  // over 4000 334 and 313; 256 over 450 257 and 242.
  const int xcd = blockIdx.x % 8, j = blockIdx.x / 8;
  if constexpr (RW == 0) {
    const int pair = blockIdx.x * 4 + wave, b = pair / a.kv_heads, kh = pair - b * a.kv_heads;
    q = load_seq(a, b, Sh::ROWS);
    if (q.mbs == 0) return;
    at = kh * (q.tiles + Sh::COST);
    stop = at + q.tiles + Sh::COST;
    w = 0;
  } else if (a.direct) {
    const int mbs = Sh::MANY ? a.most_mbs : 1, pair = j / mbs * 8 + xcd, b = pair / a.kv_heads, kh = pair - b * a.kv_heads;
    q = load_seq(a, b, Sh::ROWS);
    q.before = 0;
    q.mb = j - j / mbs * mbs;
    if (q.mb >= q.mbs) return;
    at = kh * (q.tiles + Sh::COST);
    stop = at + q.tiles + Sh::COST;
    w = 0;
  } else {
    Plan<Sh> plan;
    const int total = plan.total(a);
    if (total == 0) return;
    split = Split(total, gridDim.x);
    const int each = gridDim.x / 8;
    w = xcd * each + j;
    if (Sh::MANY) {  // stretches that are as far into the units of each row block
      const int mbs = min(a.most_mbs, each), per = each / mbs, round = j / mbs;
      w = round < per ? (j - round * mbs) * (8 * per) + xcd * per + round : j * 8 + xcd;
    }
    if (w >= split.n) return;
    at = split.share(w);
    stop = split.share(w + 1);
    q = plan.find(a, at);
    first64 = plan.first;
    base64 = plan.base;
  }

  const uint32_t lds = (uint32_t)(uintptr_t)(lds_void*)smem;
  // A 16-byte read serves lanes 0 - 3, 12 - 15 and 20 - 27 together (then 4 - 11, 16 -
  // 19, 28 - 31, and so in the other half): a piece of rows 0 - 3 and 12 - 15 and its
  // neighbour of rows 4 - 11.  A transposing read serves 32 lanes, two neighbouring
  // pieces of 8 rows.  Neither meets a bank twice.
  auto swz = [](int r) {
    const int r0 = r & 1, r1 = r >> 1 & 1, r2 = r >> 2 & 1, r3 = r >> 3 & 1;
    return CPR == 16 ? r2 | r0 << 1 | r1 << 2 | (r2 ^ r3) << 3 : r2 | r1 << 1 | (r2 ^ r3) << 2;
  };
  // of the DMA instructions of 16 rows (RW = 4: of this wave's)
  uint32_t voff[RW <= 1 ? NV : 1];
#pragma unroll
  for (int i = 0; i < (RW <= 1 ? NV : 1); ++i) {
    const int r = (RW <= 1 ? i : wave % NV) * RPI + lane / CPR, c = (lane % CPR) ^ swz(r);
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

  while (at < stop) {
    ConstArgs& a = fresh_args();
    if (at >= q.before + seq_units(a, q, Sh::COST)) {  // (loaded again: kept over the tiles, it would take their registers)
      Plan<Sh> plan;
      plan.mb = q.mb;
      plan.load(a, first64);
      plan.base = base64;
      q = plan.find(a, at);
      first64 = plan.first;
      base64 = plan.base;
    }
    const int units = q.tiles + Sh::COST, off = at - q.before, kh = (int)((uint32_t)off / (uint32_t)units);
    const int u0 = off - kh * units, u1 = min(units, u0 + (stop - at));
    const int x0 = at - u0 + Sh::COST;  // the unit of the item's first tile
    const int t0 = max(u0 - Sh::COST, 0), t1 = max(u1 - Sh::COST, 0);
    at += u1 - u0;
    if (t0 == t1) continue;  // its tiles are the next workgroup's
    const int mb = Sh::MANY ? q.mb : 0;
    const int rows = q.n * a.group, m0 = mb * Sh::ROWS + (RW <= 1 ? 0 : wave * 16 * NB);
    const int end = q.end;
    const char* const kbase = a.cache.k + kh * a.cache.head_bytes;
    const char* const vbase = a.cache.v + kh * a.cache.head_bytes;
    const int32_t* const table = in_memory(a.table) + q.b * a.ld_table;
    const float scale = a.scale;

    // ---- places of the next 64 tiles' rows: lane j has, of the tile first + j * STEP,
    // the byte offsets of its first and its second 16 rows (which may lie in different
    // pages) and the bytes from there to the last row that is to be read (0: none)
    constexpr int STEP = RW == 1 ? 4 : 1;
    const int mine = RW == 1 ? t0 + wave : t0;
    const int count = mine < t1 ? (t1 - mine + STEP - 1) / STEP : 0;
    uint32_t place[2], place_hi[2], reach[2];
    auto load_pages = [&](int i0) {
      ConstArgs& a = fresh_args();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int x = (mine + (i0 + lane) * STEP) * kTile + 16 * h;
        const bool in = i0 + lane < count && x < end;
        const int page = page_of(table, in ? x >> a.cache.shift : 0, a.cache.pages);
        if (in && page < 0 && kh == 0 && mb == 0 && (RW <= 1 || wave == 0) && a.index_errors) atomicAdd(in_memory(a.index_errors), 1);
        const bool there = in && page >= 0;
        const uint64_t at = there ? (uint64_t)page * (uint64_t)a.cache.page_bytes +
                                        (uint64_t)((uint32_t)(x & ((1 << a.cache.shift) - 1)) * a.cache.row_bytes)
                                  : 0;
        place[h] = (uint32_t)at;
        place_hi[h] = (uint32_t)(at >> 32);
        reach[h] = there ? (uint32_t)min(end - x, 16) * a.cache.row_bytes : 0;
      }
    };
    place[0] = place[1] = place_hi[0] = place_hi[1] = reach[0] = reach[1] = 0;
    if (end > 0) load_pages(0);

    // ---- this lane's rows: their queries (of a negative scale: their negatives)
    Frag qf[NB][KC];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int m = min(m0 + 16 * i + col, rows - 1);
      const int node = (int)((uint32_t)m / (uint32_t)a.group), head = kh * a.group + (m - node * a.group);
      const char* const src = in_memory(a.q) + (int64_t)(q.first + node) * a.q_token_bytes + head * a.q_head_bytes;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const int piece = 4 * c + g;
        u32x4 f = reinterpret_cast<const u32x4*>(src)[min(piece, a.hd8 - 1)];
        if (piece >= a.hd8) f = u32x4{0, 0, 0, 0};
        f ^= a.flip;
        qf[i][c] = __builtin_bit_cast(Frag, f);
      }
    }
    if (kh == 0 && mb == 0 && t0 == 0 && (RW == 0 ? lane : threadIdx.x) == 0 && a.index_errors && end < q.ctx + q.n) atomicAdd(in_memory(a.index_errors), 1);

    // halves of tile i with nothing to read, for want of a page or past the end: bits 0
    // and 1
    auto empty = [&](int i) {
      return (__builtin_amdgcn_readlane((int)reach[0], i & 63) == 0 ? 1 : 0) |
             (__builtin_amdgcn_readlane((int)reach[1], i & 63) == 0 ? 2 : 0);
    };
    // descriptor of the 16 rows of tile i's half h
    auto half_range = [&](const char* base, int i, int h) __attribute__((always_inline)) {
      const uint32_t lo = __builtin_amdgcn_readlane((int)place[h], i & 63), hi = __builtin_amdgcn_readlane((int)place_hi[h], i & 63);
      const uint32_t bytes = __builtin_amdgcn_readlane((int)reach[h], i & 63);
      const uint64_t p = (uint64_t)(uintptr_t)base + ((uint64_t)hi << 32 | lo);
      return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)p), (uint32_t)__builtin_amdgcn_readfirstlane((int)(p >> 32)) & 0xffffu,
                   i < count ? bytes : 0, 0x00020000u};
    };
    // tile i's keys (or values) to LDS byte `to`
    auto copy = [&](const char* base, int i, uint32_t to) __attribute__((always_inline)) {
      if constexpr (RW <= 1) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x4 r = half_range(base, i, h);
#pragma unroll
          for (int u = 0; u < NV; ++u) copy16(r, voff[u], to + (h * NV + u) * 1024);
        }
      } else {
        static_assert(NK == 4 || NK == 8, "a wave copies one or two pieces of a tile");
#pragma unroll
        for (int u = 0; u < NK / 4; ++u)
          copy16(half_range(base, i, NK == 8 ? u : wave >> 1), voff[0], to + (wave + 4 * u) * 1024);
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
    // the nodes that this lane's row i sees, of the tile from position x on: bit k for
    // key k (a tile of the c tokens has them all)
    auto visible = [&](int i, int x, int none) {
      int m = min(m0 + 16 * i + col, rows - 1);
      asm volatile("" : "+v"(m));  // computed here, not kept over the tiles that need none of it
      ConstArgs& a = fresh_args();
      const int node = (int)((uint32_t)m / (uint32_t)a.group);
      const uint64_t bits = a.mask ? in_memory(a.mask)[q.first + node] : ~0ull >> (63 - node);
      const int d = x - q.ctx;  // the tile's first key as a node
      uint32_t keys = d >= 64 ? 0u : d >= 0 ? (uint32_t)(bits >> d) : d <= -32 ? ~0u : (uint32_t)(bits << -d) | ((1u << -d) - 1);
      if (end - x < 32) keys &= (1u << max(end - x, 0)) - 1;
      return keys & ~((none & 1 ? 0xffffu : 0u) | (none & 2 ? 0xffff0000u : 0u));
    };
    // weights p of n tiles' scores s, the rows' offsets and sums
    auto softmax = [&](auto n, f32x4 (*s)[NB][2], Frag (*p)[NB]) __attribute__((always_inline)) {
      constexpr int N = decltype(n)::value;
      float top[NB];
      bool moves = false;
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        top[i] = -INFINITY;
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
          for (int j = 0; j < 8; ++j) top[i] = fmaxf(top[i], s[u][i][j >> 2][j & 3]);
        top[i] *= scale;
        moves |= top[i] > m_off[i] + kLazy;
      }
      if (__any(moves)) {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const float m = fmaxf(m_off[i], column_max(top[i]));
          const float keep = m_off[i] == m ? 1.f : __builtin_amdgcn_exp2f(m_off[i] - m);
          m_off[i] = m;
          l[i] *= keep;
#pragma unroll
          for (int h = 0; h < HT; ++h) o[i][h] *= keep;
        }
      }
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const float base = m_off[i] == -INFINITY ? 0.f : kLift<T> == 0.f ? -m_off[i] : kLift<T> - m_off[i];
          float e[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) e[j] = __builtin_amdgcn_exp2f(fmaf(s[u][i][j >> 2][j & 3], scale, base));
          p[u][i] = Mfma<T>::pack(e);
          // sums of the rounded weights, those that the product uses
          l[i] = Mfma<T>::sum8(p[u][i], l[i]);
        }
    };
    auto hide = [&](f32x4 (&s)[NB][2], const uint32_t (&keys)[NB]) {
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const uint32_t mine = keys[i] >> (4 * g);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          s[i][j >> 2][j & 3] = mine >> (16 * (j >> 2) + (j & 3)) & 1 ? s[i][j >> 2][j & 3] : -INFINITY;
      }
    };
    // Infinities and NaN among a tile's values: a weight of zero would not keep them
    // from a row that does not see them.  They are added to the rows that do, and
    // the product finds zeros in their place.  (Tiles of the c tokens need none of
    // this: every row sees those.)
    auto bad_values = [&](const char* vt) -> uint32_t {
      int row = lane >> 1;
      asm volatile("" : "+v"(row));
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
    auto add_bad = [&](const char* vt, uint32_t bad, const uint32_t (&keys)[NB]) {
      for (; bad; bad &= bad - 1) {
        const int k = __ffs(bad) - 1;
        const int sw = swz(k & 15);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const bool seen = keys[i] >> k & 1;
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
      int row = lane >> 1;
      asm volatile("" : "+v"(row));
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
    auto values = [&](const char* vt, int h) {
      typedef short v4s __attribute__((ext_vector_type(4)));
      typedef short v8s __attribute__((ext_vector_type(8)));
      const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(vt + vaddr[h]));
      const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(vt + vaddr[h] + 16 * RB));
      const v8s both = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
      return __builtin_bit_cast(Frag, both);
    };
    auto product = [&](int h, const Frag& vf, const Frag (&p)[NB]) {
#pragma unroll
      for (int i = 0; i < NB; ++i) o[i][h] = Mfma16<T>::mma(vf, p[i], o[i][h]);
    };
    auto products = [&](const char* vt, const Frag (&p)[NB]) {
#pragma unroll
      for (int h = 0; h < HT; ++h) product(h, values(vt, h), p);
    };

    // Tiles of the c tokens, which every row sees whole, run a loop without any of the
    // masks' work, up to one without a page; the others a second one.
    const int plain = min(max((q.ctx / kTile - mine + STEP - 1) / STEP, 0), count);
    int lost[NST];  // empty() of tile i and those behind it
    if constexpr (RW <= 1) {
      const uint32_t ring = lds + wave * (NST * 2 * TB);
      char* const mem = smem + wave * (NST * 2 * TB);
#pragma unroll
      for (int s = 0; s < NST; ++s) {
        copy(kbase, s, ring + s * 2 * TB);
        copy(vbase, s, ring + s * 2 * TB + TB);
        lost[s] = empty(s);
      }
      auto step = [&](int i, auto hides) __attribute__((always_inline)) {
        const int slot = i % NST * (2 * TB);
        char* const kt = mem + slot;
        char* const vt = kt + TB;
        f32x4 sc[NB][2];
        Frag p[NB];
        const int none = lost[0];
        if (((i + NST) & 63) == 0 && i + NST < count) load_pages(i + NST);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NK * (2 * NST - 1)) : "memory");
        scores(kt, sc);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        copy(kbase, i + NST, ring + slot);
#pragma unroll
        for (int j = 0; j + 1 < NST; ++j) lost[j] = lost[j + 1];
        lost[NST - 1] = empty(i + NST);
        uint32_t keys[NB];
        if constexpr (decltype(hides)::value) {
#pragma unroll
          for (int u = 0; u < NB; ++u) keys[u] = visible(u, (mine + i * STEP) * kTile, none);
          hide(sc, keys);
        }
        softmax(std::integral_constant<int, 1>{}, &sc, &p);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NK * (2 * NST - 1)) : "memory");
        if constexpr (decltype(hides)::value) {
          const uint32_t bad = bad_values(vt);
          if (bad) {
            add_bad(vt, bad, keys);
            clear_bad(vt);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          }
        }
        products(vt, p);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        copy(vbase, i + NST, ring + slot + TB);
      };
      int i = 0;
      for (; i < plain && lost[0] == 0; ++i) step(i, std::false_type{});
      for (; i < count; ++i) step(i, std::true_type{});
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if constexpr (RW == 1) {
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
      }
    } else {
      constexpr int NI = SUB * 2 * ((NK + 3) / 4);  // a wave's DMA instructions of a stage
      // tiles i .. i + SUB - 1 to stage st, and their empty halves
      auto fetch = [&](int i, int st) __attribute__((always_inline)) {
        int none = 0;
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
          copy(kbase, i + u, lds + (st * SUB + u) * 2 * TB);
          copy(vbase, i + u, lds + (st * SUB + u) * 2 * TB + TB);
          none |= empty(i + u) << (2 * u);
        }
        return none;
      };
#pragma unroll
      for (int s = 0; s < NST - 1; ++s) lost[s] = fetch(s * SUB, s);
      int st = 0;
      auto step = [&](int i, auto hides) __attribute__((always_inline)) {
        const int none = lost[0], ahead = i + (NST - 1) * SUB;
        if ((ahead & 63) == 0 && ahead < count) load_pages(ahead);
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(NI * (NST - 2)) : "memory");
        lost[NST - 1] = fetch(ahead, st == 0 ? NST - 1 : st - 1);
#pragma unroll
        for (int j = 0; j < NST - 1; ++j) lost[j] = lost[j + 1];
        auto keys_at = [&](int u) { return smem + (st * SUB + u) * 2 * TB; };
        if constexpr (!decltype(hides)::value) {
          // a stage's scores together: longer runs of the matrix unit, one look at the
          // rows' offsets
          f32x4 sc[SUB][NB][2];
          Frag p[SUB][NB];
#pragma unroll
          for (int u = 0; u < SUB; ++u) scores(keys_at(u), sc[u]);
          softmax(std::integral_constant<int, SUB>{}, sc, p);
#pragma unroll
          for (int u = 0; u < SUB; ++u) products(keys_at(u) + TB, p[u]);
        } else {
          for (int u = 0; u < SUB && i + u < count; ++u) {
            char* const kt = keys_at(u);
            char* const vt = kt + TB;
            f32x4 sc[NB][2];
            Frag p[NB];
            scores(kt, sc);
            uint32_t keys[NB];
#pragma unroll
            for (int j = 0; j < NB; ++j) keys[j] = visible(j, (mine + i + u) * kTile, none >> (2 * u));
            hide(sc, keys);
            softmax(std::integral_constant<int, 1>{}, &sc, &p);
            const uint32_t bad = bad_values(vt);  // the same in every wave
            if (bad) {
              add_bad(vt, bad, keys);
              asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
              if (wave == 0) clear_bad(vt);
              asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            }
            products(vt, p);
          }
        }
        st = st == NST - 1 ? 0 : st + 1;
      };
      int i = 0;
      for (; i + SUB <= plain && lost[0] == 0; i += SUB) step(i, std::false_type{});
      for (; i < count; i += SUB) step(i, std::true_type{});
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }

    // ---- the rows, or their sums for who comes last
    ConstArgs& z = fresh_args();
    const __amdgpu_buffer_rsrc_t parts = wave_rsrc(z.parts, (int64_t)2 * gridDim.x * Sh::PART * 4);
    // where row m goes
    auto out_row = [&](int m) {
      const int node = (int)((uint32_t)m / (uint32_t)z.group);
      return reinterpret_cast<T*>(in_memory(z.out) + (int64_t)(q.first + node) * z.out_bytes) +
             (int64_t)(kh * z.group + m - node * z.group) * (8 * z.hd8);
    };
    // four elements of a row, of the weighted and of the weights' sum; zeros if there is
    // no weight (weights of zero may have met values that are not finite)
    auto result = [&](const f32x4& y, bool none, float inv) {
      return Quad<T>::from(none ? make_float4(0, 0, 0, 0) : make_float4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv));
    };
    const bool whole = t0 == 0 && t1 == q.tiles;
    const int part = 2 * w + (t0 == 0 ? 1 : 0);  // a stretch ends in the first part of an item at most once
    if (RW != 1 || wave == 0) {
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int m = m0 + 16 * i + col, r = m - mb * Sh::ROWS;
        const float sum = column_sum(l[i]);
        if (m >= rows) continue;
        if (whole) {
          T* const dst = out_row(m);
          const bool none = sum == 0.f;
          const float inv = 1.0f / sum;
#pragma unroll
          for (int h = 0; h < HT; ++h)
            if (2 * h < z.hd8) *reinterpret_cast<typename Quad<T>::raw*>(dst + 16 * h + 4 * g) = result(o[i][h], none, inv);
        } else {
#pragma unroll
          for (int h = 0; h < HT; ++h)
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o[i][h]), parts,
                                                   4 * (part * Sh::PART + r * HD + 16 * h + 4 * g), 0, kThrough);
          if (g == 0)
            __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(m_off[i]), __float_as_uint(sum)}, parts,
                                                  4 * (part * Sh::PART + Sh::ROWS * HD + 2 * r), 0, kThrough);
        }
      }
    }
    if (RW == 0 || whole) continue;

    // ---- the last of eight joins them, until the item is whole
    const int w0 = split.holder(x0);
    const int stretches = split.holder(x0 + q.tiles - 1) - w0 + 1;
    auto part_of = [&](int z) { return 2 * (w0 + z) + (z == 0 ? 1 : 0); };  // of stretch z
    const int live = min(rows - mb * Sh::ROWS, Sh::ROWS);
    // Joins n sums, of stretches first, first + span, ...: into the rows if that is
    // all of the item, else in the place of the first.  L lanes a row; where rows
    // leave lanes free, `shares` groups of lanes take the stretches in turn.  Of many rows,
    // the fewer the stretches the more are asked for together (Q of them for N
    // stretches): 17 sequences over up to 12239, 4 to 10 nodes, 16 heads of 128 to a key
    // head, 105 us with one row of each lane at a time, 95 so; 64-node trees over 1000
    // to 8192 204 and 201.  Fewer rows gain nothing, and lose 1 to 4% by the longer code.
    constexpr int L = HD / 4, GROUPS = 256 / L;
    int wide = GROUPS;
    while (wide / 2 >= live) wide /= 2;
    const int shares = GROUPS / wide, group = threadIdx.x / L, c0 = threadIdx.x % L * 4, share = group / wide;
    auto join_parts = [&](auto most, auto together, int first, int span, int n, bool whole) __attribute__((always_inline)) {
      constexpr int N = decltype(most)::value, Q = decltype(together)::value;
      for (int r0 = group % wide; r0 - group % wide < live; r0 += wide * Q) {
        u32x2 ml[Q][N];
        u32x4 v[Q][N];
#pragma unroll
        for (int u = 0; u < N; ++u) {
          const int p = part_of(first + min(share + u * shares, n - 1) * span);
          if (u * shares < n) {
#pragma unroll
            for (int k = 0; k < Q; ++k) {
              const int r = min(r0 + k * wide, live - 1);
              ml[k][u] = __builtin_amdgcn_raw_buffer_load_b64(parts, 4 * (p * Sh::PART + Sh::ROWS * HD + 2 * r), 0, kCoherent);
              v[k][u] = __builtin_amdgcn_raw_buffer_load_b128(parts, 4 * (p * Sh::PART + r * HD + c0), 0, kCoherent);
            }
          }
        }
#pragma unroll
        for (int k = 0; k < Q; ++k) {
          const int r = r0 + k * wide;
          float top = -INFINITY, sum = 0.f;
          f32x4 y = {0, 0, 0, 0};
          auto add = [&](float m2, float l2, f32x4 v2) {
            const float t = fmaxf(top, m2);
            const float f1 = top == t ? 1.f : __builtin_amdgcn_exp2f(top - t), f2 = m2 == t ? 1.f : __builtin_amdgcn_exp2f(m2 - t);
            top = t;
            sum = sum * f1 + l2 * f2;
            y = y * f1 + v2 * f2;
          };
#pragma unroll
          for (int u = 0; u < N; ++u)
            if (share + u * shares < n)
              add(__uint_as_float(ml[k][u][0]), __uint_as_float(ml[k][u][1]), __builtin_bit_cast(f32x4, v[k][u]));
          if (Q == 1 && shares > 1) {  // (then one round of rows)
            f32x4* const so = reinterpret_cast<f32x4*>(smem);
            float2* const sm = reinterpret_cast<float2*>(smem + 4096);
            so[threadIdx.x] = y;
            sm[threadIdx.x] = make_float2(top, sum);
            __syncthreads();
            if (share == 0)
              for (int u = 1; u < min(shares, n); ++u) {
                const int other = threadIdx.x + u * wide * L;
                add(sm[other].x, sm[other].y, so[other]);
              }
            __syncthreads();
          }
          if (share != 0 || r >= live) continue;
          if (whole) {
            if (c0 < 8 * z.hd8)
              *reinterpret_cast<typename Quad<T>::raw*>(out_row(mb * Sh::ROWS + r) + c0) = result(y, sum == 0.f, 1.0f / sum);
          } else {
            const int p = part_of(first);
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, y), parts, 4 * (p * Sh::PART + r * HD + c0), 0, kThrough);
            if (c0 == 0)
              __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(top), __float_as_uint(sum)}, parts,
                                                    4 * (p * Sh::PART + Sh::ROWS * HD + 2 * r), 0, kThrough);
          }
        }
      }
    };
    int* const word = reinterpret_cast<int*>(smem);
    for (int span = 1, level = 0; span < stretches; span *= kJoin, ++level) {
      // stretches first, first + span, ... of this group hold its sums
      const int first = (w - w0) / (span * kJoin) * (span * kJoin);
      const int n = min(kJoin, (stretches - first + span - 1) / span);
      if (n > 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this one's sums are in memory
        __syncthreads();
        if (threadIdx.x == 0) {
          int* const counter = in_memory(z.counters) + level * (2 * gridDim.x) + part_of(first);
          const bool last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1;
          if (last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          *word = last;
        }
        __syncthreads();
        const bool joins = *word != 0;
        __syncthreads();
        if (!joins) break;
        const bool all = span * kJoin >= stretches;
        typedef std::integral_constant<int, 1> One;
        if (!Sh::MANY || shares > 1) join_parts(std::integral_constant<int, kJoin>{}, One{}, first, span, n, all);
        else if constexpr (Sh::MANY) {
          if (n <= 2) join_parts(std::integral_constant<int, 2>{}, std::integral_constant<int, 8>{}, first, span, n, all);
          else if (n <= 4) join_parts(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{}, first, span, n, all);
          else join_parts(std::integral_constant<int, kJoin>{}, std::integral_constant<int, 16 / kJoin>{}, first, span, n, all);
        }
      }
    }
  }
}

// ---------------------------------------------------------------- variants

// Workgroups of a launch: the CUs times those that a CU holds.
constexpr int kCus = 256;

template <int HD_, int NB_, int RW_, int NST_, int OCC_, int SUB_ = 1>
struct Variant {
  static constexpr int HD = HD_, NB = NB_, RW = RW_, NST = NST_, OCC = OCC_, SUB = SUB_;
  typedef TreeShape<HD, NB, RW, NST, SUB> Sh;
  static constexpr int GRID = kCus * OCC;
  static constexpr size_t BYTES = TJK_TREE_COUNTERS + (size_t)2 * GRID * Sh::PART * sizeof(float);
  static_assert(GRID <= kJoin * kJoin * kJoin && 3 * 2 * GRID * 4 <= TJK_TREE_COUNTERS && BYTES < 0x7fffffff, "counters and 32-bit offsets");
};

// Calls f with the variant for a head_dim and the rows of the largest tree: up to 64
// rows, one, two or four blocks of 16 that each of the four waves holds whole (33 to 48
// rows hold a block of none), above that waves with rows of their own that share the
// tiles (64 rows of 128 so: 105 to 108 us either way at 16 x 2000 to 4000 tokens, 16 key
// heads; of 64: 60 and 62).
template <typename F>
static auto with_variant(int head_dim, int rows, F&& f) {
  if (head_dim <= 64) {
    if (rows <= 16) return f(Variant<64, 1, 1, 2, 2>{});
    if (rows <= 32) return f(Variant<64, 2, 1, 2, 2>{});
    if (rows <= 64) return f(Variant<64, 4, 1, 2, 2>{});
    if (rows <= 128) return f(Variant<64, 2, 4, 2, 2, 2>{});
    return f(Variant<64, 4, 4, 2, 2, 2>{});
  }
  if (rows <= 16) return f(Variant<128, 1, 1, 1, 2>{});
  if (rows <= 32) return f(Variant<128, 2, 1, 1, 2>{});
  if (rows <= 64) return f(Variant<128, 4, 1, 2, 1>{});
  return f(Variant<128, 2, 4, 2, 2, 2>{});
}

// Whether each item is one workgroup's, with no plan and no joining: by the tiles of
// the longest context that the block table holds, the lengths being on the device.
// A workgroup takes about 0.3 us a tile, plan and joining 5 to 10 us.  Bounds at which
// both take as long, contexts spread from an eighth of the table up, us whole / split:
// 8 items of 32 tiles 12 / 11, 32 items 12 / 14 (head_dim 64) and 15 / 17 (128), of 63
// tiles 19 / 15 and 22 / 19; 128 items of 63 tiles 21 / 19 and 23 / 25; 256 items of 65
// tiles 23 / 28; 512 items of 63 tiles 39 / 41 and 67 / 71, of 125 tiles 67 / 65 and
// 118 / 118.
static bool whole_items(int64_t items, int64_t tiles) {
  return tiles <= std::min<int64_t>(std::max<int64_t>(32, 24 + items / 4), 96);
}

// Whether a wave has an item for itself: where there are more items than workgroups at
// once and few tiles for four waves.  us by workgroups / by waves, contexts spread from an
// eighth of the table up, head_dim 64 (128): 512 items of 8 tiles 11.6 / 12.1 (15.0 / 14.7),
// of 16 14.6 / 16.6 (20.3 / 21.3); 1024 of 2 14.5 / 8.3 (17.9 / 11.0), of 16 22.7 / 19.5
// (39.1 / 38.0), of 32 38.9 / 37.5 (65.7 / 67.6); 8192 of 2 93 / 29 (119 / 47), of 16 149 /
// 114 (228 / 213).
static bool one_wave(int64_t items, int64_t tiles, int64_t groups) { return items > groups && tiles <= 24; }

template <typename T, int HD, int NB, int RW, int NST, int OCC, int SUB>
static void start_tree(const TreeArgs& a, int64_t groups, hipStream_t s) {
  tree_attention_kernel<T, HD, NB, RW, NST, OCC, SUB><<<(unsigned)groups, 256, 0, s>>>(a);
}

template <typename T, typename V>
static int launch_tree(TreeArgs a, hipStream_t s) {
  constexpr int ROWS = V::Sh::ROWS;
  a.most_mbs = (a.max_nodes * a.group + ROWS - 1) / ROWS;
  const int64_t items = (int64_t)a.batch * a.kv_heads * a.most_mbs, tiles = (a.room + kTile - 1) / kTile;
  if (items * (std::max<int64_t>(tiles, 1) + V::Sh::COST) > INT32_MAX - kMinUnits || items > INT32_MAX / 256)
    return fail(TJK_EUNSUPPORTED, "tjk_tree_attention: the batch's sequences, heads and table are too large");
  const int64_t hd2 = 16 * a.hd8, heads = (int64_t)a.kv_heads * a.group;
  if (rows_meet(StridedRows(a.q, hd2).by(a.q_token_bytes, a.tokens).by(a.q_head_bytes, heads),
                StridedRows(a.out, heads * hd2).by(a.out_bytes, a.tokens)))
    return fail(TJK_EINVAL, "tjk_tree_attention: out may not be q, which other workgroups still read, or overlap it");
  a.direct = whole_items(items, tiles);
  if constexpr (V::RW == 1) {
    if (a.direct && one_wave(items, tiles, V::GRID)) {
      start_tree<T, V::HD, V::NB, 0, V::NST, V::OCC, V::SUB>(a, (items + 3) / 4, s);
      return check_launch("tjk_tree_attention");
    }
  }
  // whole items: eight key heads, an XCD each, and their row blocks
  const int64_t groups = a.direct ? ((int64_t)a.batch * a.kv_heads + 7) / 8 * 8 * a.most_mbs : V::GRID;
  start_tree<T, V::HD, V::NB, V::RW, V::NST, V::OCC, V::SUB>(a, groups, s);
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
  if (const int bad = check_cache(who, cache, false)) return bad;
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
  const int64_t room = std::min<int64_t>(table_cols * cache->page_size, INT32_MAX - 128);
  // (a scale of zero would make no number of what is hidden, -inf)
  const TreeArgs a{static_cast<const char*>(q), 2 * ld_q_token, 2 * ld_q_head, paged(*cache), block_table, ld_table, ctx_lens,
                   cu_nodes, tree_mask, static_cast<char*>(out), 2 * ld_out, std::max(std::fabs(scale) * log2e, FLT_MIN),
                   static_cast<int*>(workspace), reinterpret_cast<float*>(static_cast<char*>(workspace) + TJK_TREE_COUNTERS), index_errors, scale < 0 ? 0x80008000u : 0u, (int)room, (int)tokens, batch,
                   cache->kv_heads, heads / cache->kv_heads, cache->head_dim / 8, max_nodes, 0, 0};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return with_variant(cache->head_dim, max_nodes * a.group, [&](auto v) {
    return cache->dtype == TJK_F16 ? launch_tree<f16, decltype(v)>(a, s) : launch_tree<bf16, decltype(v)>(a, s);
  });
}

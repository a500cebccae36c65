// Block-scaled e4m3 GEMM: C = epi(sum_b sa[m, b] sw[n / 128, b] P_b[m, n] +
// bias), P_b the product over the b-th block of 128 along K.
//
// One v_mfma_f32_16x16x128_f8f6f4 contracts a whole block, so P_b of 16 x 16
// outputs is one instruction with a zero addend (its scale operands are left
// at 1) and the two scales cost one fp32 FMA per output and block,
// acc += P_b (sa sw).  W is the first operand, so a lane holds four
// consecutive columns of one row: the row's scale is one register per 16
// rows, and the weights' scale is the same for the whole wave (its columns lie
// in one block of 128).
#pragma once

#include "f8_common.h"
#include "gemm_tiles.h"

namespace tjk {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct F8GemmArgs {
  const uint8_t* a;
  int64_t lda;
  const float* as;
  int64_t ld_as;
  const uint8_t* w;
  int64_t ldw;
  const float* ws;
  int64_t ld_ws;
  const void* bias;
  void* c;
  int64_t ldc;
  float* cs;
  int64_t ld_cs;
  int m, n, k;
};

// In inline asm, volatile, so that the products and the FMAs that read them
// stay in the order written: as a builtin the compiler put each FMA right behind
// its product, which then waited out the matrix pipe.  The compiler does not see
// an MFMA here and inserts no wait states: 12 have to lie between the MFMA (8
// passes) and a read of its result on gfx950.
__device__ __forceinline__ void f8_mma(f32x4& d, const i32x8& w, const i32x8& a) {
  asm volatile("v_mfma_f32_16x16x128_f8f6f4 %0, %1, %2, 0" : "=&v"(d) : "v"(w), "v"(a));
}

// Chunk of a 128-byte tile row: the 16-byte chunk c of row r lies at
// c ^ f8_swz(r).  A fragment read takes chunk q or q + 4 of 16 rows in 4 lane
// groups.  Bits 0, 1, 2 of the row map to independent masks, and so do 1, 2, 3, and 2,
// 3 with mask 1: 8 rows x 1 chunk, 16 x 1 over two rows of banks and 16 x 2 over
// four all hit different banks, whichever of them the LDS serves at once.
__device__ __forceinline__ int f8_swz(int r) {
  return ((r & 1) << 2) ^ ((r >> 1) & 1) ^ (((r >> 2) & 1) << 1) ^ (((r >> 3) & 1) << 2);
}

// lds_dma16 at voff + soff.
__device__ __forceinline__ void lds_dma16_at(u32x4 rsrc, uint32_t voff, uint32_t soff, uint32_t lds_addr) {
  asm volatile("buffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voff), "s"(rsrc), "s"(soff), "{m0}"(lds_addr));
}

// One LDS DMA of 4 bytes per lane: lane's word at voff of the descriptor's
// range (zero past it) to LDS byte lds_addr + 4 * lane.
__device__ __forceinline__ void lds_dma4(u32x4 rsrc, uint32_t voff, uint32_t lds_addr) {
  asm volatile("buffer_load_dword %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "{m0}"(lds_addr));
}

// WM x WN waves of (16 MT) x (16 NT) outputs, KG groups of them along K
// (group g takes K tiles g, g + KG, ...), each with a ring of STAGES K tiles
// of 128 and a table of the scales of 16 K tiles.
template <int MT_, int NT_, int WM_, int WN_, int KG_, int STAGES_>
struct F8Geom {
  static constexpr int MT = MT_, NT = NT_, WM = WM_, WN = WN_, KG = KG_, STAGES = STAGES_;
  static constexpr int NW = WM * WN, THREADS = 64 * NW * KG;
  static constexpr int BM = 16 * MT * WM, BN = 16 * NT * WN;
  static constexpr int DA = BM / (8 * NW), DW = BN / (8 * NW), NDMA = DA + DW;  // DMA instructions per wave per K tile
  static constexpr int STAGE = (BM + BN) * 128;
  static constexpr int TAB = STAGES * STAGE;         // byte of the row scales, [16][BM]
  static constexpr int TABW = TAB + 16 * BM * 4;     // byte of the weight scales, [2][8 blocks][8]
  static constexpr int GROUP = TABW + 512;           // bytes per K group
  static constexpr int PARTS = (KG - 1) * BM * BN * 4;  // K groups' sums, over the rings
  static constexpr int LDS = KG * GROUP > PARTS ? KG * GROUP : PARTS;
  static constexpr int GP = NT % 4 == 0 ? 2 : 1;     // 16-column tiles whose W fragments are held at once
  static constexpr int NG = NT / GP;
  static_assert(DA * 8 * NW == BM && DW * 8 * NW == BN, "tile rows must split over the waves");
  static_assert(NW % 2 == 0, "row parity of the DMA instructions");
  static_assert(NG % 2 == 0 && MT % 2 == 0, "fragment double buffer; 32-row epilogue blocks");
  static_assert(128 % (16 * NT) == 0, "a wave's columns lie in one block");
  static_assert(STAGES >= 2 && STAGES <= 8, "a chunk of scales lands within 8 K tiles");
  static_assert((STAGES - 1) * NDMA + DA + 1 <= 63, "vmcnt range");
  static_assert(LDS <= 160 * 1024, "LDS");
};

// acc += the block-scaled product for this wave's (16 MT) x (16 NT) outputs
// of the tile at (m0, n0).  On return every DMA has landed and the workgroup
// has met at a barrier.
//
// Tiles reach LDS by DMA, rows of 128 bytes with the 16-byte chunk c of row r
// at c ^ f8_swz(r).  Lane (l16, q) of a fragment reads chunks q and q + 4 of row
// l16: any assignment of K to lanes is right that both operands share.
//
// Pipeline: the FMAs of a product run behind the third MFMA after it, four
// per MFMA, so none waits for the matrix pipe (and 15 instructions lie between).
// Fragments of the next GP tiles of W are read one group ahead.  Before the last
// group of a K tile everything of it is in registers: there the waves meet, the
// tile's slot is handed to the DMA of tile it + STAGES, and each A fragment is
// replaced by the next tile's as soon as its last MFMA is issued.
template <typename G>
__device__ __forceinline__ void f8_accumulate(char* smem, const F8GemmArgs& p, int m0, int n0,
                                              f32x4 (&acc)[G::NT][G::MT]) {
  constexpr int MT = G::MT, NT = G::NT, NW = G::NW, KG = G::KG, S = G::STAGES, GP = G::GP, NG = G::NG;
  const int lane = threadIdx.x & 63;
  const int gw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = gw / NW, wave = gw % NW, wm = wave / G::WN, wn = wave % G::WN;
  const int l16 = lane & 15, q16 = lane >> 4;
  char* const gsm = smem + kg * G::GROUP;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)gsm;
  const int nkt = (p.k + 127) / 128, nit = (nkt + KG - 1) / KG;

  // rows past M (N) lie outside the buffer ranges and arrive as zeros
  const u32x4 rsa = lds_dma_rsrc(p.a + (int64_t)m0 * p.lda, (int64_t)min(G::BM, p.m - m0) * p.lda);
  const u32x4 rsw = lds_dma_rsrc(p.w + (int64_t)n0 * p.ldw, (int64_t)min(G::BN, p.n - n0) * p.ldw);
  const u32x4 rsas = lds_dma_rsrc(p.as + (int64_t)m0 * p.ld_as, (int64_t)min(G::BM, p.m - m0) * p.ld_as * 4);
  const int nb0 = n0 / 128, nbs = (p.n + 127) / 128;
  const u32x4 rsws = lds_dma_rsrc(p.ws + (int64_t)nb0 * p.ld_ws, (int64_t)(nbs - nb0) * p.ld_ws * 4);

  // DMA instruction i fills rows (i NW + wave) 8 .. + 7; lane l lands in row
  // l / 8, physical chunk l % 8.  NW is even, so the chunk is the same for all.
  // A lane's offset stays the same over the K tiles, whose own offset is a
  // scalar: it takes no vector instruction next to the FMAs.
  const int line0 = wave * 8 + lane / 8;
  const uint32_t lcb = (uint32_t)(((lane & 7) ^ f8_swz(line0)) << 4);
  uint32_t voff[G::NDMA];
#pragma unroll
  for (int i = 0; i < G::NDMA; ++i)
    voff[i] = i < G::DA ? (uint32_t)(line0 + 8 * NW * i) * (uint32_t)p.lda + lcb
                        : (uint32_t)(line0 + 8 * NW * (i - G::DA)) * (uint32_t)p.ldw + lcb;
  auto dma = [&](int it, int i) __attribute__((always_inline)) {
    const uint32_t slot = lds0 + (uint32_t)(it % S) * G::STAGE;
    const uint32_t dst = slot + (i < G::DA ? (i * NW + wave) * 1024 : G::BM * 128 + ((i - G::DA) * NW + wave) * 1024);
    lds_dma16_at(i < G::DA ? rsa : rsw, voff[i], (uint32_t)(it * KG + kg) * 128u, dst);
  };
  // Called before the DMA of K tile `it`: from the K tile that is not whole on,
  // the chunks past K lie outside the buffer ranges, from the first one past
  // the end on all do (they arrive as zeros).
  auto past_end = [&](int it) __attribute__((always_inline)) {
    const uint32_t out = (uint32_t)(it * KG + kg) * 128u + lcb < (uint32_t)p.k ? 0u : kPastEnd;
#pragma unroll
    for (int i = 0; i < G::NDMA; ++i) voff[i] |= out;
  };
  // scales of K tiles 8 c .. 8 c + 7 of this group, into half c & 1 of the table
  auto scale_dma = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < G::DA; ++d) {
      const int f0 = (d * NW + wave) * 64, f = f0 + lane, i = f / G::BM, row = f % G::BM;
      const int kt = (8 * c + i) * KG + kg;
      const uint32_t off = kt < nkt ? ((uint32_t)row * (uint32_t)p.ld_as + (uint32_t)kt) * 4u : kPastEnd;
      lds_dma4(rsas, off, lds0 + G::TAB + (c & 1) * 8 * G::BM * 4 + f0 * 4);
    }
    if (wave == 0) {
      const int nb = lane >> 3, kt = (8 * c + (lane & 7)) * KG + kg;
      const uint32_t off = kt < nkt ? ((uint32_t)nb * (uint32_t)p.ld_ws + (uint32_t)kt) * 4u : kPastEnd;
      lds_dma4(rsws, off, lds0 + G::TABW + (c & 1) * 256);
    }
  };

  const int sw = (q16 ^ f8_swz(l16)) << 4;
  const char* const fa0 = gsm + (wm * 16 * MT + l16) * 128;
  const char* const fw0 = gsm + G::BM * 128 + (wn * 16 * NT + l16) * 128;
  auto frag = [&](const char* rows) __attribute__((always_inline)) {
    const i32x4 lo = *reinterpret_cast<const i32x4*>(rows + sw), hi = *reinterpret_cast<const i32x4*>(rows + (sw ^ 64));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  const float* const tab = reinterpret_cast<const float*>(gsm + G::TAB) + wm * 16 * MT + l16;
  const float* const tabw = reinterpret_cast<const float*>(gsm + G::TABW) + ((n0 + wn * 16 * NT) / 128 - nb0) * 8;

  // The rows of A of K tile it are all in registers by its second group, where
  // a second meeting (MEET) hands their part of the slot to the DMA of tile
  // it + S, so that the DMA spreads over the K tile: A's over the groups in the
  // middle, W's in the last one.
  constexpr bool MEET = NG >= 3;
  constexpr int NMID = MEET ? (NG - 2) * MT : 1;
  scale_dma(0);
#pragma unroll
  for (int t = 0; t < S; ++t) {
    past_end(t);
#pragma unroll
    for (int i = 0; i < G::NDMA; ++i) dma(t, i);
  }
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 1) * G::NDMA) : "memory");
  asm volatile("s_barrier" ::: "memory");

  i32x8 fa[MT], fw[2][GP];
  f32x4 part[4];
  float raw[MT], raw_w, s[MT], s_last[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    fa[j] = frag(fa0 + j * 2048);
    raw[j] = tab[16 * j];
    s_last[j] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < GP; ++i) fw[0][i] = frag(fw0 + i * 2048);
  raw_w = tabw[0];
#pragma unroll
  for (int j = 0; j < MT; ++j) s[j] = raw[j] * raw_w;
#pragma unroll
  for (int v = 0; v < 4; ++v) part[v] = f32x4{0.f, 0.f, 0.f, 0.f};

  // Product v of a K tile: group v / (MT GP), 16-row tile j, W tile i.  The FMAs
  // of the product three back (of the previous K tile for v < 3).
  constexpr int TILES = MT * NT;
  static_assert(TILES % 4 == 0, "ring of four products");
  auto join = [&](int v, const float (&f)[MT]) __attribute__((always_inline)) {
    f32x4& p4 = part[v & 3];
    asm volatile("" : "+v"(p4));  // not before the MFMAs above
    const int j = v % (MT * GP) / GP;
    f32x4& c = acc[v / (MT * GP) * GP + v % GP][j];
#pragma unroll
    for (int r = 0; r < 4; ++r) c[r] = fmaf(p4[r], f[j], c[r]);
  };

  for (int it = 0; it < nit; ++it) {
    const int st = (it % S) * G::STAGE, nx = ((it + 1) % S) * G::STAGE;
    if ((it & 7) == 0) scale_dma((it >> 3) + 1);
    if (((it + S) * KG + kg + 1) * 128 > p.k) past_end(it + S);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const bool last = g + 1 == NG;
      if (last) {
        // tile it + 1 landed
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S - 2) * G::NDMA + (MEET ? G::DA : 0)) : "memory");
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
      } else if (MEET && g == 1) {
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int j = 0; j < MT; ++j) {
#pragma unroll
        for (int i = 0; i < GP; ++i) {
          const int v = (g * MT + j) * GP + i;
          f8_mma(part[v & 3], fw[g & 1][i], fa[j]);
          if (v < 3) join(v + TILES - 3, s_last);
          else join(v - 3, s);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (last) {
          if (j == 0) {
            const int o = (it + 1) & 15;
#pragma unroll
            for (int jj = 0; jj < MT; ++jj) raw[jj] = tab[o * G::BM + 16 * jj];
            raw_w = tabw[(o >> 3) * 64 + (o & 7)];
          }
          fa[j] = frag(fa0 + nx + j * 2048);
          if (j < GP) fw[0][j] = frag(fw0 + nx + j * 2048);
          constexpr int D0 = MEET ? G::DA : 0, ND = G::NDMA - D0;
#pragma unroll
          for (int d = j * ND / MT; d < (j + 1) * ND / MT; ++d) dma(it + S, D0 + d);
        } else if (j < GP) {
          fw[(g + 1) & 1][j] = frag(fw0 + st + ((g + 1) * GP + j) * 2048);
        }
        if (MEET && g >= 1 && !last) {
          const int u = (g - 1) * MT + j;
#pragma unroll
          for (int d = u * G::DA / NMID; d < (u + 1) * G::DA / NMID; ++d) dma(it + S, d);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      s_last[j] = s[j];
      s[j] = raw[j] * raw_w;
    }
  }
  asm volatile("s_nop 7\n\ts_nop 3" : "+v"(part[1]), "+v"(part[2]), "+v"(part[3]));
#pragma unroll
  for (int v = TILES - 3; v < TILES; ++v) join(v, s_last);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// Adds the K groups' sums in group order into group 0's accumulators, through
// LDS.  True for the waves that hold the result.
template <typename G>
__device__ __forceinline__ bool f8_join_groups(char* smem, f32x4 (&acc)[G::NT][G::MT]) {
  if constexpr (G::KG > 1) {
    const int gw = threadIdx.x >> 6, kg = gw / G::NW, lane = threadIdx.x & 63;
    constexpr int TILES = G::MT * G::NT;
    float4* const base = reinterpret_cast<float4*>(smem) + (gw % G::NW) * TILES * 64 + lane;
    constexpr int STEP = G::NW * TILES * 64;
    if (kg > 0) {
#pragma unroll
      for (int i = 0; i < G::NT; ++i)
#pragma unroll
        for (int j = 0; j < G::MT; ++j)
          base[(kg - 1) * STEP + (i * G::MT + j) * 64] = __builtin_bit_cast(float4, acc[i][j]);
    }
    __syncthreads();
    if (kg == 0) {
#pragma unroll
      for (int o = 0; o < G::KG - 1; ++o)
#pragma unroll
        for (int i = 0; i < G::NT; ++i)
#pragma unroll
          for (int j = 0; j < G::MT; ++j)
            acc[i][j] += __builtin_bit_cast(f32x4, base[o * STEP + (i * G::MT + j) * 64]);
    }
    __syncthreads();
    return kg == 0;
  } else {
    return true;
  }
}

// Internal epilogue modes: the output in e4m3 with scales per row and 128
// columns, after the bias (and GELU).
constexpr int kEpiF8 = 8, kEpiF8Gelu = 9;

// e4m3 output of a wave's (16 MT) x (16 NT) outputs at (mw, nw).  Lane (l16,
// q) holds columns 16 i + 4 q .. + 3 of rows 16 j + l16, so a row's largest
// magnitude over the wave's columns takes two lane exchanges; where a block of
// 128 columns spans several waves they trade theirs through LDS (`red`, BM x WN
// floats; every wave of the workgroup calls this).  Words are put in rows through
// `stage` (16 MT x 16 NT bytes of the wave's own), the 16-byte piece i of row r
// at i ^ x(r), and leave as whole pieces.
template <bool GELU, typename G>
__device__ __forceinline__ void f8_epilogue(const F8GemmArgs& p, f32x4 (&acc)[G::NT][G::MT], int mw, int nw, int wm,
                                            int wn, int lane, bool holds, float* red, char* stage) {
  constexpr int MT = G::MT, NT = G::NT, WPB = 128 / (16 * NT);
  const int l16 = lane & 15, q16 = lane >> 4;
  float top[MT];
  if (holds) {
    const float* const bias = static_cast<const float*>(p.bias);
    float4 b[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) b[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (bias != nullptr) {
#pragma unroll
      for (int i = 0; i < NT; ++i) b[i] = *reinterpret_cast<const float4*>(bias + min(nw + 16 * i + 4 * q16, p.n - 4));
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      top[j] = 0.f;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        f32x4 v = acc[i][j];
        v[0] += b[i].x; v[1] += b[i].y; v[2] += b[i].z; v[3] += b[i].w;
        const bool in = nw + 16 * i + 4 * q16 < p.n;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (GELU) v[r] = gelu_erf(v[r]);
          top[j] = fmaxf(top[j], in ? fabsf(v[r]) : 0.f);
        }
        acc[i][j] = v;
      }
      top[j] = fmaxf(top[j], __shfl_xor(top[j], 16));
      top[j] = fmaxf(top[j], __shfl_xor(top[j], 32));
    }
  }
  if constexpr (WPB > 1) {
    if (holds && q16 == 0) {
#pragma unroll
      for (int j = 0; j < MT; ++j) red[wn * G::BM + wm * 16 * MT + 16 * j + l16] = top[j];
    }
    __syncthreads();
    if (holds) {
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int o = 0; o < WPB; ++o)
          top[j] = fmaxf(top[j], red[(wn / WPB * WPB + o) * G::BM + wm * 16 * MT + 16 * j + l16]);
    }
  }
  if (!holds) return;
  auto x = [](int r) { return NT >= 8 ? r & 7 : (r >> 1) & (NT - 1); };
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const float s = f8_scale(top[j]), inv = __builtin_amdgcn_rcpf(s);
    const int m = mw + 16 * j + l16;
    if (q16 == 0 && wn % WPB == 0 && m < p.m && nw < p.n) p.cs[(int64_t)m * p.ld_cs + nw / 128] = s;
#pragma unroll
    for (int i = 0; i < NT; ++i)
      *reinterpret_cast<uint32_t*>(stage + (16 * j + l16) * 16 * NT + ((i ^ x(l16)) << 4) + 4 * q16) =
          f8_pack4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3], inv);
  }
  uint8_t* const c = static_cast<uint8_t*>(p.c);
  const bool a16 = ((uintptr_t)c & 15) == 0 && p.ldc % 16 == 0;
  constexpr int NPC = 16 * MT * NT;
#pragma unroll
  for (int it = 0; it < NPC / 64; ++it) {
    const int pc = lane + 64 * it, r = pc / NT, i = pc % NT;
    const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 16 * NT + ((i ^ x(r & 15)) << 4));
    const int m = mw + r, n = nw + 16 * i;
    if (m < p.m && n < p.n) {
      uint8_t* const o = c + (int64_t)m * p.ldc + n;
      if (a16 && n + 16 <= p.n) {
        *reinterpret_cast<uint4*>(o) = v;
      } else {  // N and ldc are multiples of 4
        reinterpret_cast<uint32_t*>(o)[0] = v.x;
        if (n + 4 < p.n) reinterpret_cast<uint32_t*>(o)[1] = v.y;
        if (n + 8 < p.n) reinterpret_cast<uint32_t*>(o)[2] = v.z;
        if (n + 12 < p.n) reinterpret_cast<uint32_t*>(o)[3] = v.w;
      }
    }
  }
}

// T: the bias's type, and the output's unless that is e4m3
template <typename T, int EPI, typename G>
__global__ __launch_bounds__(G::THREADS, G::THREADS >= 512 ? 2 : 1) void gemm_f8_kernel(F8GemmArgs p) {
  __shared__ __align__(16) char smem[G::LDS];
  int pid_m, pid_n;
  tile_coords(blockIdx.x, (p.m + G::BM - 1) / G::BM, (p.n + G::BN - 1) / G::BN, pid_m, pid_n);
  const int m0 = pid_m * G::BM, n0 = pid_n * G::BN;
  f32x4 acc[G::NT][G::MT];
#pragma unroll
  for (int i = 0; i < G::NT; ++i)
#pragma unroll
    for (int j = 0; j < G::MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  f8_accumulate<G>(smem, p, m0, n0, acc);
  const bool holds = f8_join_groups<G>(smem, acc);
  const int lane = threadIdx.x & 63;
  const int gw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = gw % G::NW;
  const int wm = wave / G::WN, wn = wave % G::WN;
  const int mw = m0 + wm * 16 * G::MT, nw = n0 + wn * 16 * G::NT;
  if constexpr (EPI == kEpiF8 || EPI == kEpiF8Gelu) {
    constexpr int RED = G::BM * G::WN * 4;
    f8_epilogue<EPI == kEpiF8Gelu, G>(p, acc, mw, nw, wm, wn, lane, holds, reinterpret_cast<float*>(smem),
                                      smem + RED + wave * 256 * G::MT * G::NT);
  } else {
    constexpr int FM = G::MT / 2, FN = G::NT / 2;
    static_assert(EpiStage<T, EPI, FN>::BYTES * G::NW <= G::LDS, "epilogue staging");
    if (holds)
      epilogue<T, EPI, FM, FN, NoPrefetch, kResBatch, true>(acc, static_cast<const T*>(p.bias), p.c, p.ldc, p.m, p.n,
                                                            mw, nw, lane, smem + wave * EpiStage<T, EPI, FN>::BYTES);
  }
}

}  // namespace tjk

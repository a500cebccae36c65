// Block-scaled e4m3 GEMM: C = epi(sum_b sa[m, b] sw[n / 128, b] P_b[m, n] +
// bias), P_b the product over the b-th block of 128 along K.
//
// Two v_mfma_f32_32x32x64_f8f6f4 contract a block: P_b of 32 x 32 outputs
// starts from a zero addend and takes the two scales as one fp32 FMA per output
// and block, acc += P_b (sa sw).  W is the first operand, so a lane holds four
// consecutive columns of one row: the row's scale is one register per 32 rows,
// and the weights' scale is the same for the whole wave (its columns lie in one
// block of 128).
//
// What bounds it: an f8f6f4 MFMA keeps the vector issue of its SIMD for 16
// cycles, whatever its shape (it reads 16 operand registers), a vector
// instruction for 4; measured with loops of nothing else.  With 16 x 16 x 128 MFMAs
// (32 cycles each) the four FMAs that belong to one fill the rest of it, and
// every address or scale instruction more delays the matrix unit.  With 32 x 32 x 64
// (64 cycles) the eight FMAs leave four issue slots.
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

// The product of one block.  In inline asm, volatile, so that the products and
// the FMAs that read them stay in the order written: as a builtin the compiler
// put each FMA right behind its product, which then waited out the matrix pipe.
// The compiler does not see an MFMA here and inserts no wait states: 20 have to
// lie between the second MFMA (16 passes) and a read of its result on gfx950.
__device__ __forceinline__ void f8_mma(f32x16& d, const i32x8 (&w)[2], const i32x8 (&a)[2]) {
  asm volatile(
      "v_mfma_f32_32x32x64_f8f6f4 %0, %1, %3, 0\n\t"
      "v_mfma_f32_32x32x64_f8f6f4 %0, %2, %4, %0\n\t"
      "s_nop 1"
      : "=&v"(d)
      : "v"(w[0]), "v"(w[1]), "v"(a[0]), "v"(a[1]));
}

// Chunk of a 128-byte tile row: the 16-byte chunk c of row r lies at
// c ^ f8_swz(r).  A fragment read takes one chunk of 32 rows in each lane half.
// Row bits 0, 1, 2 map to independent masks, and so do 1, 2, 3, and 2, 3, 4: 8
// rows, 16 over two rows of banks and 32 over four all hit different banks,
// whichever of them the LDS serves at once.  Measured: no conflicts.
__device__ __forceinline__ int f8_swz(int r) {
  return ((r & 1) << 1) ^ ((r & 2) << 1) ^ ((r >> 2) & 1) ^ (((r >> 3) & 1) << 1) ^ (((r >> 4) & 1) << 2);
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

// W x W waves of (32 FM) x (32 FN) outputs, KG groups of them along K (group g
// takes K tiles g, g + KG, ...).  A K tile (128 deep) is PPS panels: panel j <
// FM of A holds every wave row's j-th 32 rows, panel FM + i of W every wave
// column's i-th 32 columns.  Each group has a ring of R panels and a table of the
// scales of 8 K tiles.
template <int FM_, int FN_, int W_, int KG_, int R_>
struct F8Geom {
  static constexpr int FM = FM_, FN = FN_, W = W_, KG = KG_, R = R_;
  static constexpr int NW = W * W, THREADS = 64 * NW * KG;
  static constexpr int WTM = 32 * FM, WTN = 32 * FN, BM = WTM * W, BN = WTN * W;
  static constexpr int PPS = FM + FN, PANEL = 32 * W * 128;
  static constexpr int DP = 4 / W, ND = PPS * DP;  // DMA instructions per wave: of a panel, of a K tile
  static constexpr int DS = 2 * FM / W;            // of the row scales of four K tiles
  static constexpr int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }
  static constexpr int PHASES = R / gcd(R, PPS);   // K tiles until the ring's slots repeat
  static constexpr int TAB = R * PANEL;            // byte of the row scales, [8][BM]
  static constexpr int TABW = TAB + 8 * BM * 4;    // byte of the weight scales, [2][16 blocks][4]
  static constexpr int GROUP = TABW + 512;         // bytes per K group
  static constexpr int PARTS = (KG - 1) * BM * BN * 4;  // K groups' sums, over the rings
  static constexpr int LDS = KG * GROUP > PARTS ? KG * GROUP : PARTS;
  static_assert(W == 1 || W == 2, "4 / W DMA instructions per panel");
  static_assert(FN % 2 == 0, "fragment double buffer, ring of two products");
  static_assert(128 % WTN == 0, "a wave's columns lie in one block");
  static_assert(DS * W == 2 * FM, "scales must split over the waves");
  static_assert(R >= PPS + FM + 1 && PHASES <= 4, "the panels that are read together fit beside those of a K tile");
  static_assert(R * DP + ND <= 63, "vmcnt range");
  static_assert(LDS <= 160 * 1024, "LDS");
};

// acc += the block-scaled product for this wave's (32 FM) x (32 FN) outputs
// of the tile at (m0, n0).  On return every DMA has landed and the workgroup
// has met at a barrier.
//
// Panels reach LDS by DMA, rows of 128 bytes with the 16-byte chunk c of row r
// at c ^ f8_swz(r).  Lane (l32, hi) of a fragment's half h reads chunks
// 4 h + hi and 4 h + 2 + hi of row l32: any assignment of K to lanes is right
// that both operands share.
//
// Pipeline.  A K tile runs as FN W tiles of FM products.  The FMAs of a product
// run behind the two MFMAs of the next one, so none waits for the matrix pipe (18
// instructions and a pause of two lie between).  Fragments are read one W tile
// ahead: W's i + 1 during tile i, and during the last one A's and W's first of
// the next K tile, each A fragment in place of the one whose last MFMA has been
// issued.  Panels are read in the order A0 .. W0 W1 .. of each K tile, so the ring
// is a queue: at the meeting before a W tile the panels read during the one
// before are free, and those about to be read have landed.  A K tile's ND DMA
// instructions, each into the slot of a panel read at least one meeting ago, are
// spread evenly over its products: a burst stalls the waves that issue it.
template <typename G>
__device__ __forceinline__ void f8_accumulate(char* smem, const F8GemmArgs& p, int m0, int n0,
                                              f32x16 (&acc)[G::FN][G::FM]) {
  constexpr int FM = G::FM, FN = G::FN, NW = G::NW, KG = G::KG, R = G::R, PPS = G::PPS, DP = G::DP;
  const int lane = threadIdx.x & 63;
  const int gw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = gw / NW, wave = gw % NW, wm = wave / G::W, wn = wave % G::W;
  const int l32 = lane & 31, hi = lane >> 5;
  char* const gsm = smem + kg * G::GROUP;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)gsm;
  const int nkt = (p.k + 127) / 128, nit = (nkt + KG - 1) / KG;

  // rows past M (N) lie outside the buffer ranges and arrive as zeros
  const u32x4 rsa = lds_dma_rsrc(p.a + (int64_t)m0 * p.lda, (int64_t)min(G::BM, p.m - m0) * p.lda);
  const u32x4 rsw = lds_dma_rsrc(p.w + (int64_t)n0 * p.ldw, (int64_t)min(G::BN, p.n - n0) * p.ldw);
  const u32x4 rsas = lds_dma_rsrc(p.as + (int64_t)m0 * p.ld_as, (int64_t)min(G::BM, p.m - m0) * p.ld_as * 4);
  const int nb0 = n0 / 128, nbs = (p.n + 127) / 128;
  const u32x4 rsws = lds_dma_rsrc(p.ws + (int64_t)nb0 * p.ld_ws, (int64_t)(nbs - nb0) * p.ld_ws * 4);

  // DMA instruction d of a panel fills its rows (d NW + wave) 8 .. + 7: with
  // two wave rows instruction d the d-th one's.  Lane l lands in row l / 8,
  // physical chunk l % 8.  A lane's offset stays the same over the K tiles, whose
  // own offset is a scalar: it takes no vector instruction next to the FMAs.
  uint32_t voff[PPS][DP];
  auto dma_chunk = [&](int d) __attribute__((always_inline)) {
    return (uint32_t)(((lane & 7) ^ f8_swz((d * NW + wave) * 8 + lane / 8)) << 4);
  };
#pragma unroll
  for (int y = 0; y < PPS; ++y)
#pragma unroll
    for (int d = 0; d < DP; ++d) {
      const int r = (d * NW + wave) * 8 + lane / 8;
      const int row = y < FM ? r / 32 * G::WTM + y * 32 + r % 32 : r / 32 * G::WTN + (y - FM) * 32 + r % 32;
      voff[y][d] = (uint32_t)row * (uint32_t)(y < FM ? p.lda : p.ldw) + dma_chunk(d);
    }
  // instruction d of panel y of K tile `it` into a slot
  auto dma = [&](int it, int y, int d, int slot) __attribute__((always_inline)) {
    lds_dma16_at(y < FM ? rsa : rsw, voff[y][d], (uint32_t)(it * KG + kg) * 128u,
                 lds0 + slot * G::PANEL + (d * NW + wave) * 1024);
  };
  // Called before the DMA of panel y of K tile `it`: from the K tile that is not
  // whole on, the chunks past K lie outside the buffer ranges, from the first
  // one past the end on all do (they arrive as zeros).
  auto past_end = [&](int it, int y) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < DP; ++d)
      voff[y][d] |= (uint32_t)(it * KG + kg) * 128u + dma_chunk(d) < (uint32_t)p.k ? 0u : kPastEnd;
  };
  // scales of K tiles 4 c .. 4 c + 3 of this group, into half c & 1 of the table
  auto scale_dma = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < G::DS; ++d) {
      const int f0 = (d * NW + wave) * 64, f = f0 + lane, i = f / G::BM, row = f % G::BM;
      const int kt = (4 * c + i) * KG + kg;
      const uint32_t off = kt < nkt ? ((uint32_t)row * (uint32_t)p.ld_as + (uint32_t)kt) * 4u : kPastEnd;
      lds_dma4(rsas, off, lds0 + G::TAB + (c & 1) * 4 * G::BM * 4 + f0 * 4);
    }
    if (wave == 0) {
      const int nb = lane >> 2, kt = (4 * c + (lane & 3)) * KG + kg;
      const uint32_t off = kt < nkt ? ((uint32_t)nb * (uint32_t)p.ld_ws + (uint32_t)kt) * 4u : kPastEnd;
      lds_dma4(rsws, off, lds0 + G::TABW + (c & 1) * 256);
    }
  };

  const int sw = (hi ^ f8_swz(l32)) << 4;
  const char* const fa0 = gsm + (wm * 32 + l32) * 128;
  const char* const fw0 = gsm + (wn * 32 + l32) * 128;
  auto frag = [&](const char* rows, int slot, int h) __attribute__((always_inline)) {
    const i32x4 lo = *reinterpret_cast<const i32x4*>(rows + (sw ^ (h * 64)) + slot * G::PANEL);
    const i32x4 up = *reinterpret_cast<const i32x4*>(rows + (sw ^ (h * 64 + 32)) + slot * G::PANEL);
    return __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  const float* const tab = reinterpret_cast<const float*>(gsm + G::TAB) + wm * G::WTM + l32;
  const float* const tabw = reinterpret_cast<const float*>(gsm + G::TABW) + ((n0 + wn * G::WTN) / 128 - nb0) * 4;

  scale_dma(0);
#pragma unroll
  for (int q = 0; q < R; ++q) {
    past_end(q / PPS, q % PPS);
#pragma unroll
    for (int d = 0; d < DP; ++d) dma(q / PPS, q % PPS, d, q);
  }
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"((R - FM - 1) * DP) : "memory");
  asm volatile("s_barrier" ::: "memory");

  i32x8 fa[FM][2], fw[2][2];
  f32x16 part[2];
  float raw[FM], raw_w, s[FM], s_last = 0.f;
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    fa[j][0] = frag(fa0, j, 0);
    fa[j][1] = frag(fa0, j, 1);
    raw[j] = tab[32 * j];
  }
  fw[0][0] = frag(fw0, FM, 0);
  fw[0][1] = frag(fw0, FM, 1);
  raw_w = tabw[0];
#pragma unroll
  for (int j = 0; j < FM; ++j) s[j] = raw[j] * raw_w;
#pragma unroll
  for (int r = 0; r < 16; ++r) part[1][r] = 0.f;

  // The FMAs of product v = i FM + j (the last of the K tile before: v = -1).
  constexpr int TILES = FM * FN;
  auto join = [&](int v, float f) __attribute__((always_inline)) {
    f32x16& d = part[v & 1];
    asm volatile("" : "+v"(d));  // not before the MFMAs above
    f32x16& c = acc[(v + TILES) % TILES / FM][(v + TILES) % FM];
#pragma unroll
    for (int r = 0; r < 16; ++r) c[r] = fmaf(d[r], f, c[r]);
  };

  // One K tile, its panels in slots PH PPS .. (mod R).
  auto step = [&](auto PH, int it) __attribute__((always_inline)) {
    constexpr int q0 = decltype(PH)::value * PPS;
    if ((it & 3) == 0) scale_dma((it >> 2) + 1);
    if (((it + (PPS - 1 + R) / PPS) * KG + kg + 1) * 128 > p.k) {
#pragma unroll
      for (int y = 0; y < PPS; ++y) past_end(it + (y + R) / PPS, (y + R) % PPS);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      const bool last = i + 1 == FN;
      // Landed: the panels read during this W tile; in flight at most what was
      // issued after them.
      constexpr int ISSUED = R * DP;  // before this K tile, from its own first panel on
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(ISSUED + i * FM * G::ND / TILES -
                                                         DP * (last ? PPS + FM + 1 : FM + i + 2))
                   : "memory");
      asm volatile("s_barrier" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        const int v = i * FM + j;
        f8_mma(part[v & 1], fw[i & 1], fa[j]);
        if (last) {
          if (j == 0) {
            const int o = (it + 1) & 7;
#pragma unroll
            for (int jj = 0; jj < FM; ++jj) raw[jj] = tab[o * G::BM + 32 * jj];
            raw_w = tabw[(o >> 2) * 64 + (o & 3)];
          }
          fa[j][0] = frag(fa0, (q0 + PPS + j) % R, 0);
          fa[j][1] = frag(fa0, (q0 + PPS + j) % R, 1);
        }
        // fragments of the next W tile, a half after each product
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (j == min(h, FM - 1)) fw[(i + 1) & 1][h] = frag(fw0, (q0 + FM + (last ? PPS : i + 1)) % R, h);
#pragma unroll
        for (int d = v * G::ND / TILES; d < (v + 1) * G::ND / TILES; ++d)
          dma(it + (d / DP + R) / PPS, (d / DP + R) % PPS, d % DP, (q0 + d / DP) % R);
        join(v - 1, v == 0 ? s_last : s[(v - 1) % FM]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    s_last = s[FM - 1];
#pragma unroll
    for (int j = 0; j < FM; ++j) s[j] = raw[j] * raw_w;
  };
  for (int it = 0; it < nit;) {
    step(IntC<0>{}, it);
    if (++it >= nit) break;
    if constexpr (G::PHASES > 1) {
      step(IntC<1>{}, it);
      if (++it >= nit) break;
    }
    if constexpr (G::PHASES > 2) {
      step(IntC<2>{}, it);
      if (++it >= nit) break;
    }
    if constexpr (G::PHASES > 3) {
      step(IntC<3>{}, it);
      ++it;
    }
  }
  asm volatile("s_nop 15\n\ts_nop 3" : "+v"(part[1]));
  join(-1, s_last);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// Adds the K groups' sums in group order into group 0's accumulators, through
// LDS.  True for the waves that hold the result.
template <typename G>
__device__ __forceinline__ bool f8_join_groups(char* smem, f32x16 (&acc)[G::FN][G::FM]) {
  if constexpr (G::KG > 1) {
    const int gw = threadIdx.x >> 6, kg = gw / G::NW, lane = threadIdx.x & 63;
    constexpr int QUADS = G::FM * G::FN * 4;  // of a lane
    float4* const base = reinterpret_cast<float4*>(smem) + (gw % G::NW) * QUADS * 64 + lane;
    constexpr int STEP = G::NW * QUADS * 64;
    if (kg > 0) {
#pragma unroll
      for (int i = 0; i < G::FN; ++i)
#pragma unroll
        for (int j = 0; j < G::FM; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            base[(kg - 1) * STEP + ((i * G::FM + j) * 4 + q) * 64] =
                make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
    }
    __syncthreads();
    if (kg == 0) {
#pragma unroll
      for (int o = 0; o < G::KG - 1; ++o)
#pragma unroll
        for (int i = 0; i < G::FN; ++i)
#pragma unroll
          for (int j = 0; j < G::FM; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float4 v = base[o * STEP + ((i * G::FM + j) * 4 + q) * 64];
              acc[i][j][4 * q] += v.x; acc[i][j][4 * q + 1] += v.y;
              acc[i][j][4 * q + 2] += v.z; acc[i][j][4 * q + 3] += v.w;
            }
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

// e4m3 output of a wave's (32 FM) x (32 FN) outputs at (mw, nw).  Lane (l32,
// hi) holds columns 32 i + 8 g + 4 hi .. + 3 of rows 32 j + l32, so a row's
// largest magnitude over the wave's columns takes one lane exchange; where a
// block of 128 columns spans several waves they trade theirs through LDS (`red`,
// BM x W floats; every wave of the workgroup calls this).  Words are put in rows
// through `stage` (1024 FM FN bytes of the wave's own), the 16-byte piece c of
// row r at c ^ x(r), and leave as whole pieces.
template <bool GELU, typename G>
__device__ __forceinline__ void f8_epilogue(const F8GemmArgs& p, f32x16 (&acc)[G::FN][G::FM], int mw, int nw, int wm,
                                            int wn, int lane, bool holds, float* red, char* stage) {
  constexpr int FM = G::FM, FN = G::FN, WPB = 128 / G::WTN;
  const int l32 = lane & 31, hi = lane >> 5;
  float top[FM];
  if (holds) {
    const float* const bias = static_cast<const float*>(p.bias);
    float4 b[FN][4];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) b[i][g] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (bias != nullptr) {
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          b[i][g] = *reinterpret_cast<const float4*>(bias + min(nw + 32 * i + 8 * g + 4 * hi, p.n - 4));
    }
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      top[j] = 0.f;
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const bool in = nw + 32 * i + 8 * g + 4 * hi < p.n;
          const float add[4] = {b[i][g].x, b[i][g].y, b[i][g].z, b[i][g].w};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float v = acc[i][j][4 * g + r] + add[r];
            if (GELU) v = gelu_erf(v);
            acc[i][j][4 * g + r] = v;
            top[j] = fmaxf(top[j], in ? fabsf(v) : 0.f);
          }
        }
      top[j] = fmaxf(top[j], __shfl_xor(top[j], 32));
    }
  }
  if constexpr (WPB > 1) {
    if (holds && hi == 0) {
#pragma unroll
      for (int j = 0; j < FM; ++j) red[wn * G::BM + wm * G::WTM + 32 * j + l32] = top[j];
    }
    __syncthreads();
    if (holds) {
#pragma unroll
      for (int j = 0; j < FM; ++j)
#pragma unroll
        for (int o = 0; o < WPB; ++o)
          top[j] = fmaxf(top[j], red[(wn / WPB * WPB + o) * G::BM + wm * G::WTM + 32 * j + l32]);
    }
  }
  if (!holds) return;
  constexpr int LPR = 2 * FN;  // pieces per row: 8 or 4
  static_assert(LPR == 8 || LPR == 4, "staged rows of 128 or 64 bytes");
  auto x = [](int r) { return LPR == 8 ? r & 7 : (r >> 1) & 3; };
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const float s = f8_scale(top[j]), inv = __builtin_amdgcn_rcpf(s);
    const int m = mw + 32 * j + l32;
    if (hi == 0 && wn % WPB == 0 && m < p.m && nw < p.n) p.cs[(int64_t)m * p.ld_cs + nw / 128] = s;
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<uint32_t*>(stage + (32 * j + l32) * 16 * LPR + (((2 * i + (g >> 1)) ^ x(l32)) << 4) +
                                     8 * (g & 1) + 4 * hi) =
            f8_pack4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3], inv);
  }
  uint8_t* const c = static_cast<uint8_t*>(p.c);
  const bool a16 = ((uintptr_t)c & 15) == 0 && p.ldc % 16 == 0;
  constexpr int NPC = 32 * FM * LPR;
#pragma unroll
  for (int it = 0; it < NPC / 64; ++it) {
    const int pc = lane + 64 * it, r = pc / LPR, i = pc % LPR;
    const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 16 * LPR + ((i ^ x(r & 31)) << 4));
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
__global__ __launch_bounds__(G::THREADS, G::THREADS <= 256 && G::LDS > 80 * 1024 ? 1 : 2) void gemm_f8_kernel(F8GemmArgs p) {
  __shared__ __align__(16) char smem[G::LDS];
  int pid_m, pid_n;
  tile_coords(blockIdx.x, (p.m + G::BM - 1) / G::BM, (p.n + G::BN - 1) / G::BN, pid_m, pid_n);
  const int m0 = pid_m * G::BM, n0 = pid_n * G::BN;
  f32x16 acc[G::FN][G::FM];
  zero_acc<float, G::FM, G::FN>(acc);
  f8_accumulate<G>(smem, p, m0, n0, acc);
  const bool holds = f8_join_groups<G>(smem, acc);
  const int lane = threadIdx.x & 63;
  const int gw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = gw % G::NW;
  const int wm = wave / G::W, wn = wave % G::W;
  const int mw = m0 + wm * G::WTM, nw = n0 + wn * G::WTN;
  if constexpr (EPI == kEpiF8 || EPI == kEpiF8Gelu) {
    constexpr int RED = G::BM * G::W * 4;
    static_assert(RED + G::BM * G::BN <= G::LDS, "epilogue staging");
    f8_epilogue<EPI == kEpiF8Gelu, G>(p, acc, mw, nw, wm, wn, lane, holds, reinterpret_cast<float*>(smem),
                                      smem + RED + wave * 1024 * G::FM * G::FN);
  } else {
    typedef EpiStage<T, EPI, G::FN> E;
    static_assert(E::BYTES * G::NW <= G::LDS, "epilogue staging");
    if (holds)
      epilogue<T, EPI, G::FM, G::FN>(acc, static_cast<const T*>(p.bias), p.c, p.ldc, p.m, p.n, mw, nw, lane,
                                     smem + wave * E::BYTES);
  }
}

}  // namespace tjk

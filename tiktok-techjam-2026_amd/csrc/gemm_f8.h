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
// (64 cycles) the eight FMAs leave four issue slots.  One wave issues an instruction
// every 7 cycles at most, so a SIMD with one wave falls behind its products; with
// two the matrix unit is the bound, and in large launches the clock that their power
// leaves: 8192^3 takes 457 us (2.4 PFLOP/s; matrix unit busy for 66% of the cycles at
// 1.74 GHz), its MFMAs alone 290, and 412 a library product with one scale per
// tensor.  8192 x 8192 x 2048: 137 us.  Few rows are bound by the passage of the
// weights: 8 x 8192 x 2048 in 6.0 us, 2.8 TB/s, of which 2.5 us are launch, latency
// and join.
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

// The two halves of a block's product.  In inline asm, volatile, so that the
// products and the FMAs that read them stay in the order written: as a builtin the
// compiler put each FMA right behind its product, which then waited out the
// matrix pipe.  The compiler does not see an MFMA here and inserts no wait
// states: 20 have to lie between the second half (16 passes) and a read of the
// result on gfx950.
__device__ __forceinline__ void f8_mma0(f32x16& d, const i32x8& w, const i32x8& a) {
  asm volatile("v_mfma_f32_32x32x64_f8f6f4 %0, %1, %2, 0" : "=&v"(d) : "v"(w), "v"(a));
}
__device__ __forceinline__ void f8_mma1(f32x16& d, const i32x8& w, const i32x8& a) {
  asm volatile("v_mfma_f32_32x32x64_f8f6f4 %0, %1, %2, %0\n\ts_nop 1" : "+v"(d) : "v"(w), "v"(a));
}

// A fragment half (32 e4m3 values of one row per lane) in fp16, which holds
// every e4m3 value exactly (NaN stays NaN): four operands of a 32x32x16 MFMA.
__device__ __forceinline__ f16x8 f8_widen(const i32x8& f, int q) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  f16x8 w;
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    const f16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(f[2 * q + d], 1.0f, false);
    const f16x2 up = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(f[2 * q + d], 1.0f, true);
    w[4 * d] = lo[0];
    w[4 * d + 1] = lo[1];
    w[4 * d + 2] = up[0];
    w[4 * d + 3] = up[1];
  }
  return w;
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

// WM x WN waves of (32 FM) x (32 FN) outputs, KG groups of them along K (group
// g takes K tiles g, g + KG, ...).  A K tile (128 deep) is PPS panels: panel
// j < FM of A holds every wave row's j-th 32 rows, panel FM + i of W every wave
// column's i-th 32 columns.  Each group has a ring of RA panels of A, one of RW
// panels of W, and a table of the scales of 8 K tiles.  MEETINGS: bit i, the
// waves meet before the i-th W tile (0 and the last are among them).  EXACT:
// exact products, in fp16.
template <int FM_, int FN_, int WM_, int WN_, int KG_, int RA_, int RW_, int MEETINGS_ = -1, bool EXACT_ = false>
struct F8Geom {
  static constexpr bool EXACT = EXACT_;
  static constexpr int FM = FM_, FN = FN_, WM = WM_, WN = WN_, KG = KG_, RA = RA_, RW = RW_;
  static constexpr int NW = WM * WN, THREADS = 64 * NW * KG, TILES = FM * FN;
  static constexpr int WTM = 32 * FM, WTN = 32 * FN, BM = WTM * WM, BN = WTN * WN;
  static constexpr int PPS = FM + FN, PA = 32 * WM * 128, PW = 32 * WN * 128;  // panel bytes
  static constexpr int DPA = 4 / WN, DPW = 4 / WM;        // DMA instructions per wave: of a panel
  static constexpr int ND = FM * DPA + FN * DPW;          // of a K tile
  static constexpr bool SPLIT = FN < 4;                   // reads and DMA between a product's MFMAs
  static constexpr int DS = 2 * FM / WN;                  // of the row scales of four K tiles
  static constexpr int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }
  static constexpr int lcm(int a, int b) { return a / gcd(a, b) * b; }
  static constexpr int PHASES = lcm(RA / gcd(RA, FM), RW / gcd(RW, FN));  // K tiles until the slots repeat
  static constexpr int RINGW = RA * PA;                // byte of W's ring
  static constexpr int TAB = RINGW + RW * PW;          // of the row scales, [8][BM]
  static constexpr int TABW = TAB + 8 * BM * 4;        // of the weight scales, [2][16 blocks][4]
  static constexpr int GROUP = TABW + 512;             // bytes per K group
  static constexpr int PITCH = BN + 4;                 // floats between rows of the K groups' sums
  static constexpr int PARTS = KG > 1 ? KG * BM * PITCH * 4 : 0;  // which lie over the rings
  static constexpr int BIAS = KG * GROUP > PARTS ? KG * GROUP : PARTS;  // byte of the bias, as it is stored
  // No DMA past the last K tile, in workgroups whose every wave is a K group: each
  // takes few K tiles, and two past them cost 0.2 of 4.1 us (K = 512).  Not where
  // waves share K tiles: branches in the K loop cost 4 to 15% of a K tile.
  static constexpr bool TRIM = KG > 1 && NW == 1;
  // (whole LDS DMA instructions bring the bias: 64 words each, zeros past the tile)
  static constexpr int BIAS_BYTES = BN * 4 > 256 ? BN * 4 : 256;
  static constexpr int LDS = BIAS + BIAS_BYTES;

  // Panel y (A: y < FM) of a K tile: the first of its DMA instructions, their
  // number; the panel that goes into its slot when it has been read, and how many
  // K tiles later that one is.
  static constexpr int first(int y) { return y < FM ? y * DPA : FM * DPA + (y - FM) * DPW; }
  static constexpr int count(int y) { return y < FM ? DPA : DPW; }
  static constexpr int panel(int d) { return d < FM * DPA ? d / DPA : FM + (d - FM * DPA) / DPW; }
  static constexpr int next(int y) { return y < FM ? (y + RA) % FM : FM + (y - FM + RW) % FN; }
  static constexpr int ahead(int y) { return y < FM ? (y + RA) / FM : (y - FM + RW) / FN; }
  static constexpr int AHEAD = ahead(FM - 1) > ahead(PPS - 1) ? ahead(FM - 1) : ahead(PPS - 1);
  // Whether the waves meet before W tile i, and the W tile of the meeting after.
  static constexpr bool meets(int i) { return i == 0 || i == FN - 1 || (MEETINGS_ >> i & 1); }
  static constexpr int until(int i) { return i + 1 >= FN || meets(i + 1) ? i + 1 : until(i + 1); }
  static constexpr int since(int i) { return meets(i) ? i : since(i - 1); }
  // DMA instructions of a K tile issued before its product v: evenly spread, but
  // only into slots whose panel was read before the last meeting (A's and W's
  // first during the K tile before, W's i + 1 during W tile i).
  static constexpr int issued(int v) {
    return v == 0 ? 0
                  : v * ND / TILES < FM * DPA + (since((v - 1) / FM) + 1) * DPW
                        ? v * ND / TILES
                        : FM * DPA + (since((v - 1) / FM) + 1) * DPW;
  }
  // DMA instructions issued up to W tile i after those of panel y of the K tile
  // `later` K tiles on.
  static constexpr int after(int i, int y, int later) {
    for (int z = 0; z < PPS; ++z)
      if (next(z) == y) return issued(i * FM) - (later - ahead(z)) * ND - first(z) - count(z);
    return 0;
  }
  // How many may be in flight at the meeting before W tile i: what was issued
  // after the last of the panels that are read until the next meeting.
  static constexpr int in_flight(int i) {
    int n = 63;
    for (int t = i; t < until(i); ++t)
      for (int y = 0; y < PPS; ++y)
        if (t + 1 < FN ? y == FM + t + 1 : y <= FM) {
          const int a = after(i, y, t + 1 < FN ? 0 : 1);
          if (a < n) n = a;
        }
    return n;
  }
  static constexpr bool valid() {
    for (int i = 0; i < FN; ++i)
      if (meets(i) && in_flight(i) < 0) return false;
    return issued(TILES) == ND;
  }
  static_assert(DPA * WN == 4 && DPW * WM == 4, "panels must split over the waves");
  static_assert(FN % 2 == 0 || (FM == 1 && FN == 1 && PHASES % 2 == 0), "fragment double buffer, ring of two products");
  static_assert(!EXACT || (FN == 2 && FM <= 2), "two W tiles, two A fragments");
  static_assert(128 % WTN == 0, "a wave's columns lie in one block");
  static_assert(DS * WN == 2 * FM, "scales must split over the waves");
  static_assert(RA >= FM && RW >= FN && PHASES <= 4, "rings of whole K tiles at least");
  static_assert(valid(), "panels land before they are read");
  static_assert(RA / FM * FM * DPA + RW / FN * FN * DPW + 2 * ND <= 63, "vmcnt range");
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
// Pipeline.  A K tile runs as FN W tiles of FM products of two MFMAs (64 cycles
// each).  The FMAs of a product run behind the second MFMA of the next one, so none
// waits for the matrix pipe (18 instructions and a pause of two lie between).
// Between the MFMAs (SPLIT) or behind them come the fragment reads and the DMA
// instructions; a DMA that cannot issue yet stalls its wave, and each takes 16 cycles
// of the CU, so four waves that issue one at once hold each other up for 64: under
// the first MFMA that costs nothing.  1024 x 1024 x 4096 in 128 x 128 tiles, one
// wave per SIMD: 19.2 us, against 21.4 behind both; the tiles of four W tiles have
// no registers for it (they spilled, 133 -> 143 us at 8192 x 8192 x 2048).
// Fragments are read one W tile
// ahead: W's i + 1 during tile i, and during the last one A's and W's first of
// the next K tile, each A fragment in place of the one whose last MFMA has been
// issued.  At a meeting of the waves the panels read since the last one are free,
// and those about to be read have landed.  A K tile's ND DMA instructions, each
// into the slot of a panel read before the last meeting, are spread over its
// products: a burst stalls the waves that issue it.
//
// EXACT.  The e4m3 MFMAs drop low bits of products (1.0e-5 of an output's scale
// was lost, against 1e-7 here); an e4m3 output's scales are fp32 results, so
// its sums are formed of fragments widened to fp16 in registers, 8 products of 32
// cycles in place of 2 of 64, with the same panels, rings and meetings.  Behind each
// MFMA stand two FMAs of the product before and four or eight conversions, each
// into the registers of an operand that was used for the last time: W's next tile
// behind its last row block, A's next K tile behind its last W tile and, the second
// fragment, behind the next K tile's first product (its registers are free then).
// 2048 x 1024 x 4096, one wave per SIMD: 30.1 us, against 35.0 with the conversions
// in one piece.  Two waves: 4096^3 117 us (1.17 PFLOP/s, the matrix unit busy for
// 57% of the cycles at 1.95 GHz), 5430 x 4096 x 1024 with GELU 57 us (36 with the
// e4m3 MFMAs).  With a long K or few rows a 2-byte output and quantize_f8 are quicker.
// Of a K tile there the DMA takes 16% and the conversions 18% beside the products; with
// neither it is the products' own time.
template <typename G>
__device__ __forceinline__ void f8_accumulate(char* smem, const F8GemmArgs& p, int m0, int n0,
                                              f32x16 (&acc)[G::FN][G::FM]) {
  constexpr int FM = G::FM, FN = G::FN, NW = G::NW, KG = G::KG, PPS = G::PPS;
  const int lane = threadIdx.x & 63;
  const int gw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = gw / NW, wave = gw % NW, wm = wave / G::WN, wn = wave % G::WN;
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

  // DMA instruction d of a panel fills its rows u .. u + 7, u = (d NW + wave) 8;
  // lane l lands in row u + l / 8, physical chunk l % 8.  A lane's offset stays
  // the same over the K tiles, whose own offset is a scalar: it takes no vector
  // instruction next to the FMAs.
  uint32_t voff[G::ND];
  auto dma_u = [&](int i) __attribute__((always_inline)) { return ((i - G::first(G::panel(i))) * NW + wave) * 8; };
  const int lane_chunk = (lane & 7) ^ f8_swz(lane / 8);
  auto dma_chunk = [&](int i) __attribute__((always_inline)) { return (uint32_t)((lane_chunk ^ f8_swz(dma_u(i) & 31)) << 4); };
  {
    const uint32_t ra = (uint32_t)(lane / 8) * (uint32_t)p.lda, rw = (uint32_t)(lane / 8) * (uint32_t)p.ldw;
#pragma unroll
    for (int i = 0; i < G::ND; ++i) {
      const int y = G::panel(i), u = dma_u(i);
      const uint32_t row = u / 32 * (y < FM ? G::WTM : G::WTN) + (y < FM ? y : y - FM) * 32 + u % 32;
      voff[i] = row * (uint32_t)(y < FM ? p.lda : p.ldw) + ((y < FM ? ra : rw) + dma_chunk(i));
    }
  }
  // byte in its ring of the slot that panel y of K tile ph (mod PHASES) lies in
  auto slot = [](int ph, int y) __attribute__((always_inline)) {
    return y < FM ? (ph * FM + y) % G::RA * G::PA : (ph * FN + y - FM) % G::RW * G::PW;
  };
  // DMA instruction i of K tile `it` into the slot at byte `to` of its ring
  auto dma = [&](int it, int i, int to) __attribute__((always_inline)) {
    lds_dma16_at(i < FM * G::DPA ? rsa : rsw, voff[i], (uint32_t)(it * KG + kg) * 128u,
                 lds0 + (i < FM * G::DPA ? 0 : G::RINGW) + to + ((i - G::first(G::panel(i))) * NW + wave) * 1024);
  };
  // Called before the DMA of panel y of K tile `it`: from the K tile that is not
  // whole on, the chunks past K lie outside the buffer ranges, from the first
  // one past the end on all do (they arrive as zeros).
  auto past_end = [&](int it, int y) __attribute__((always_inline)) {
#pragma unroll
    for (int i = G::first(y); i < G::first(y) + G::count(y); ++i)
      voff[i] |= (uint32_t)(it * KG + kg) * 128u + dma_chunk(i) < (uint32_t)p.k ? 0u : kPastEnd;
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
  const char* const fw0 = gsm + G::RINGW + (wn * 32 + l32) * 128;
  auto frag = [&](const char* rows, int at, int h) __attribute__((always_inline)) {
    const i32x4 lo = *reinterpret_cast<const i32x4*>(rows + (sw ^ (h * 64)) + at);
    const i32x4 up = *reinterpret_cast<const i32x4*>(rows + (sw ^ (h * 64 + 32)) + at);
    return __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  const float* const tab = reinterpret_cast<const float*>(gsm + G::TAB) + wm * G::WTM + l32;
  const float* const tabw = reinterpret_cast<const float*>(gsm + G::TABW) + ((n0 + wn * G::WTN) / 128 - nb0) * 4;

  // The panels that fill the rings, in the order in which K tiles before the
  // first would have issued them; then a wait as before the last W tile of a K
  // tile -1.
  scale_dma(0);
#pragma unroll
  for (int t = -G::AHEAD; t < 0; ++t)
#pragma unroll
    for (int z = 0; z < PPS; ++z)
      if (t + G::ahead(z) >= 0) {
        const int y = G::next(z), it = t + G::ahead(z);
        if (G::TRIM && it >= nit) continue;
        past_end(it, y);
#pragma unroll
        for (int d = 0; d < G::count(y); ++d) dma(it, G::first(y) + d, slot(it, y));
      }
  // TRIM, near the end: waits until no more than `tiles` K tiles are in flight (DMA
  // instructions land in order, K tile by K tile; of several W tiles: until all have).
  static_assert(!G::TRIM || FN > 1 || (G::ahead(0) == G::AHEAD && G::ahead(FM) == G::AHEAD && G::AHEAD <= 4),
                "the panels of a K tile are in flight together, with three more K tiles at most");
  auto wait_tiles = [&](int tiles) __attribute__((always_inline)) {
    if (FN > 1 || tiles <= 0)
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    else if (tiles == 1)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(G::ND) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * G::ND) : "memory");
  };
  if (G::TRIM && nit < G::AHEAD)
    wait_tiles(nit - 1);
  else
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(G::in_flight(FN - 1) + G::issued(G::TILES) - G::issued((FN - 1) * FM))
                 : "memory");
  if constexpr (NW > 1) asm volatile("s_barrier" ::: "memory");

  i32x8 fa[FM][2], fw[2][2];
  f32x16 part[2];
  float raw[FM], raw_w, s[FM], s_last = 0.f;
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    fa[j][0] = frag(fa0, slot(0, j), 0);
    fa[j][1] = frag(fa0, slot(0, j), 1);
    raw[j] = tab[32 * j];
  }
  fw[0][0] = frag(fw0, slot(0, FM), 0);
  fw[0][1] = frag(fw0, slot(0, FM), 1);
  raw_w = tabw[0];
#pragma unroll
  for (int j = 0; j < FM; ++j) s[j] = raw[j] * raw_w;
#pragma unroll
  for (int r = 0; r < 16; ++r) part[1][r] = 0.f;

  // The FMAs of product v = i FM + j (the last of the K tile before: v = -1), of a
  // K tile that begins with part `odd`.
  constexpr int TILES = G::TILES;
  auto join = [&](int v, int odd, float f) __attribute__((always_inline)) {
    f32x16& d = part[(v + odd) & 1];
    asm volatile("" : "+v"(d));  // not before the MFMAs above
    f32x16& c = acc[(v + TILES) % TILES / FM][(v + TILES) % FM];
#pragma unroll
    for (int r = 0; r < 16; ++r) c[r] = fmaf(d[r], f, c[r]);
  };

  f16x8 ah[G::EXACT ? FM : 1][8], wh[8];
  if constexpr (G::EXACT) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      ah[0][q] = f8_widen(fa[0][q >> 2], q & 3);
      wh[q] = f8_widen(fw[0][q >> 2], q & 3);
    }
  }

  // One K tile, PH = it mod PHASES.
  auto step = [&](auto PH, int it) __attribute__((always_inline)) {
    constexpr int ph = decltype(PH)::value;
    if ((it & 3) == 0 && (!G::TRIM || it + 4 < nit)) scale_dma((it >> 2) + 1);
    if (((it + G::AHEAD) * KG + kg + 1) * 128 > p.k) {
#pragma unroll
      for (int z = 0; z < PPS; ++z) past_end(it + G::ahead(z), G::next(z));
    }
    __builtin_amdgcn_sched_barrier(0);
    auto tile = [&](auto I) __attribute__((always_inline)) {
      constexpr int i = decltype(I)::value;
      constexpr bool last = i + 1 == FN;
      if constexpr (G::meets(i)) {
        constexpr int in_flight = G::in_flight(i);
        if (G::TRIM && it + G::AHEAD >= nit)  // fewer in flight
          wait_tiles(nit - 2 - it);
        else
          asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(in_flight) : "memory");
        if constexpr (NW > 1) asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (G::EXACT) {
        auto raw_w_half = [&](int h) __attribute__((always_inline)) {
          fw[0][h] = frag(fw0, last ? slot(ph + 1, FM) : slot(ph, FM + i + 1), h);
        };
        auto widen_w = [&](int q) __attribute__((always_inline)) {
          wh[q] = f8_widen(fw[0][q >> 2], q & 3);
          asm volatile("" : "+v"(wh[q]));
        };
        auto widen_a = [&](int j, int q) __attribute__((always_inline)) {
          ah[j][q] = f8_widen(fa[j][q >> 2], q & 3);
          asm volatile("" : "+v"(ah[j][q]));
        };
#pragma unroll
        for (int j = 0; j < FM; ++j) {
          const int v = i * FM + j;
          f32x16& d = part[v & 1];
          const f32x16& e = part[~v & 1];
          f32x16& c = acc[(v - 1 + TILES) % TILES / FM][(v - 1 + TILES) % FM];
          const float f = v == 0 ? s_last : s[(v - 1 + FM) % FM];
          if (j == 0) {
            raw_w_half(0);
            raw_w_half(1);
          }
          if (last && j == 0) {
            fa[0][0] = frag(fa0, slot(ph + 1, 0), 0);
            fa[0][1] = frag(fa0, slot(ph + 1, 0), 1);
            const int o = (it + 1) & 7;
#pragma unroll
            for (int jj = 0; jj < FM; ++jj) raw[jj] = tab[o * G::BM + 32 * jj];
            raw_w = tabw[(o >> 2) * 64 + (o & 3)];
          }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            d = __builtin_amdgcn_mfma_f32_32x32x16_f16(wh[q], ah[j][q], q ? d : f32x16{}, 0, 0, 0);
            if (q == 1 || q == 5) {  // half of the product's DMA instructions each
              const int n0 = G::issued(v), n1 = G::issued(v + 1), mid = (n0 + n1 + 1) / 2;
#pragma unroll
              for (int n = q == 1 ? n0 : mid; n < (q == 1 ? mid : n1); ++n) {
                const int z = G::panel(n), y = G::next(z);
                dma(it + G::ahead(z), G::first(y) + n - G::first(z), slot(ph, z));
              }
            }
            if (q > 0)  // not at once behind the product that they read
#pragma unroll
              for (int r = (q - 1) * 16 / 7; r < q * 16 / 7; ++r) c[r] = fmaf(e[r], f, c[r]);
            if constexpr (FM == 2) {
              if (v == 0) widen_a(1, q);
              if (j == 1) widen_w(q);
              if (last && j == 0 && q >= 4) widen_a(0, q - 4);
              if (last && j == 1 && q < 4) widen_a(0, q + 4);
              if (last && j == 1 && (q == 4 || q == 7)) fa[1][q == 7] = frag(fa0, slot(ph + 1, 1), q == 7);
            } else if (q >= 4) {
              widen_w(q - 4);
              if (last) widen_a(0, q - 4);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          if constexpr (FM == 1) {
#pragma unroll
            for (int q = 4; q < 8; ++q) {
              widen_w(q);
              if (last) widen_a(0, q);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        return;
      }
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        const int v = i * FM + j;
        constexpr int odd = TILES % 2 ? ph & 1 : 0, w = (i + odd) & 1;
        f8_mma0(part[(v + odd) & 1], fw[w][0], fa[j][0]);
        if constexpr (!G::SPLIT) f8_mma1(part[(v + odd) & 1], fw[w][1], fa[j][1]);
        __builtin_amdgcn_sched_barrier(0);
        if (last) {
          if (j == 0) {
            const int o = (it + 1) & 7;
#pragma unroll
            for (int jj = 0; jj < FM; ++jj) raw[jj] = tab[o * G::BM + 32 * jj];
            raw_w = tabw[(o >> 2) * 64 + (o & 3)];
          } else if (G::SPLIT) {
            fa[j - 1][1] = frag(fa0, slot(ph + 1, j - 1), 1);
          }
          fa[j][0] = frag(fa0, slot(ph + 1, j), 0);
          if (!G::SPLIT) fa[j][1] = frag(fa0, slot(ph + 1, j), 1);
        }
        // fragments of the next W tile, a half per product
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (j == min(h, FM - 1))
            fw[w ^ 1][h] = frag(fw0, last ? slot(ph + 1, FM) : slot(ph, FM + i + 1), h);
#pragma unroll
        for (int d = G::issued(v); d < G::issued(v + 1); ++d) {
          const int z = G::panel(d), y = G::next(z);
          if (!G::TRIM || it + G::ahead(z) < nit) dma(it + G::ahead(z), G::first(y) + d - G::first(z), slot(ph, z));
        }
        if constexpr (G::SPLIT) {
          __builtin_amdgcn_sched_barrier(0);
          f8_mma1(part[(v + odd) & 1], fw[w][1], fa[j][1]);
          if (last && j + 1 == FM) fa[j][1] = frag(fa0, slot(ph + 1, j), 1);
        }
        join(v - 1, odd, v == 0 ? s_last : s[(v - 1 + FM) % FM]);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    tile(IntC<0>{});
    if constexpr (FN > 1) tile(IntC<1>{});
    if constexpr (FN > 2) {
      tile(IntC<2>{});
      tile(IntC<3>{});
    }
    s_last = s[FM - 1];
#pragma unroll
    for (int j = 0; j < FM; ++j) s[j] = raw[j] * raw_w;
  };
#pragma unroll 1
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
  if constexpr (G::EXACT) {
    join(-1, 0, s_last);
  } else {
    if (TILES % 2 && (nit & 1)) {
      asm volatile("s_nop 15\n\ts_nop 3" : "+v"(part[0]));
      join(-1, 1, s_last);
    } else {
      asm volatile("s_nop 15\n\ts_nop 3" : "+v"(part[1]));
      join(-1, 0, s_last);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// Two values rounded to nearest even in a 2-byte type, one word.
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef T t2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), t2));
}

// The output rows of a wave, (32 FM) x (32 FN) elements of ES bytes from the
// wave-uniform (mw, nw): stores at byte offsets of a buffer range that ends with
// the last row and column, so that rows past M are dropped; columns past N go
// past the range.
struct F8Rows {
  __amdgpu_buffer_rsrc_t r;
  uint32_t pitch;
  int cols;  // columns from nw on
  template <int AUX>
  __device__ __forceinline__ void put16(int row, int col, int es, const uint4& v) const {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, at(row, col, 16 / es, es), 0, AUX);
  }
  __device__ __forceinline__ void put8(int row, int col, int es, uint32_t x, uint32_t y) const {
    __builtin_amdgcn_raw_buffer_store_b64(u32x2{x, y}, r, at(row, col, 8 / es, es), 0, 0);
  }
  __device__ __forceinline__ void put4(int row, int col, int es, uint32_t x) const {
    __builtin_amdgcn_raw_buffer_store_b32(x, r, at(row, col, 4 / es, es), 0, 0);
  }
  __device__ __forceinline__ uint32_t at(int row, int col, int n, int es) const {
    return col + n <= cols ? (uint32_t)row * pitch + (uint32_t)(col * es) : kPastEnd;
  }
};

template <typename G>
__device__ __forceinline__ F8Rows f8_rows(const F8GemmArgs& p, int mw, int nw, int es) {
  const int rows = min(G::WTM, p.m - mw), cols = min(G::WTN, p.n - nw);
  const int64_t bytes = rows > 0 && cols > 0 ? ((int64_t)(rows - 1) * p.ldc + cols) * es : 0;
  return F8Rows{wave_rsrc(static_cast<char*>(p.c) + ((int64_t)mw * p.ldc + nw) * es, bytes), (uint32_t)(p.ldc * es), cols};
}

// GELU to within 2e-6 of its own value.  gelu_erf's error is absolute, 1.5e-7 |v|,
// which is 0.4% of GELU(-4) and a quarter of GELU(-6): nothing next to a value
// of ordinary size, but an e4m3 block whose values all lie there takes its scale
// from them.  GELU(v) = max(v, 0) - u h, u = |v|, h = erfc(u / sqrt 2) / 2 =
// exp(-u^2 / 2) R(u); R as a polynomial in t = 1 / (1 + u / 4) without a constant term,
// fitted for the least largest relative error (3.2e-8) over u >= 0.  exp is the square
// of 2^-x with 2 x = u^2 log2(e) / 2 rounded, corrected by what the rounding left over:
// 2^-x is a normal number for every result that fp32 holds, 2^-2x would be flushed.
__device__ __forceinline__ float gelu_low(float v) {
  const float u = fabsf(v), t = __builtin_amdgcn_rcpf(fmaf(u, 0.25f, 1.0f));
  float r = 0.0199038982f;
  r = fmaf(r, t, -0.0814161226f);
  r = fmaf(r, t, 0.096593f);
  r = fmaf(r, t, -0.0327164568f);
  r = fmaf(r, t, 0.0642895103f);
  r = fmaf(r, t, 0.0587661937f);
  r = fmaf(r, t, 0.0816461295f);
  r = fmaf(r, t, 0.0934616029f);
  r = fmaf(r, t, 0.0997366682f);
  r = fmaf(r, t, 0.0997355655f);
  const float y = fminf(u, 32.0f);  // 0 from there on
  const float s = y * y, x2 = s * 0.72134752f;
  // what s, x2 and the constant are short of u^2 log2(e) / 2
  const float left = fmaf(fmaf(y, y, -s), 0.72134752f, fmaf(s, 9.62981517e-09f, fmaf(s, 0.72134752f, -x2)));
  const float e = __builtin_amdgcn_exp2f(-0.5f * x2);
  const float q = u * (r * t) * fmaf(left, -0.69314718f, 1.0f);
  return fmaf(-(q * e), e, fmaxf(v, 0.0f));
}

// Whether gelu_erf will not do for some values of a row: it will if `top`, the
// largest magnitude of their GELU, is at least 1 / 32 of `far`, that of the values
// themselves.  It is then off by 1.5e-7 x 32 = 4.8e-6 of `top` at most.  Values of both
// signs hardly ever get there; those that all lie below -2.2 do.  5430 x 4096 x 1024
// takes 58.2 us with this, 57.1 with gelu_erf alone and 65.4 with gelu_low for all.
__device__ __forceinline__ bool gelu_is_low(float top, float far) { return top < far * (1.0f / 32); }

// acc <- epilogue(acc + bias) of a wave's outputs; the bias of the tile's
// columns lies in LDS, in T.
template <typename T, bool GELU, bool F8, typename G>
__device__ __forceinline__ void f8_values(const char* smem, f32x16 (&acc)[G::FN][G::FM], int wn, int hi) {
  const T* const bias = reinterpret_cast<const T*>(smem + G::BIAS) + wn * G::WTN + 4 * hi;
#pragma unroll
  for (int i = 0; i < G::FN; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4 b = Quad<T>::to(*reinterpret_cast<const typename Quad<T>::raw*>(bias + 32 * i + 8 * g));
      const float add[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < G::FM; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float v = acc[i][j][4 * g + r] + add[r];
          acc[i][j][4 * g + r] = GELU && !F8 ? gelu_erf(v) : v;
        }
    }
  if constexpr (GELU && F8) {
#pragma unroll
    for (int j = 0; j < G::FM; ++j) {
      f32x16 y[G::FN];
      float top = 0.f, far = 0.f;
#pragma unroll
      for (int i = 0; i < G::FN; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          y[i][r] = gelu_erf(acc[i][j][r]);
          top = fmaxf(top, fabsf(y[i][r]));
          far = fmaxf(far, fabsf(acc[i][j][r]));
        }
      const bool low = gelu_is_low(top, far);  // of the lane's values, all in one row
      if (__any(low)) {
#pragma unroll
        for (int i = 0; i < G::FN; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) y[i][r] = low ? gelu_low(acc[i][j][r]) : y[i][r];
      }
#pragma unroll
      for (int i = 0; i < G::FN; ++i) acc[i][j] = y[i];
    }
  }
}

// Epilogue of K groups: their sums go to LDS in rows, and every thread takes
// pieces of 8 columns, adds the groups' in group order, and stores the result.
// 16 lanes hold an e4m3 block.  128 x 2048 x 512 with GELU in 32 x 64 tiles: 4.3 us,
// against 5.5 with the join and the epilogue by group 0's wave alone.
template <typename T, bool GELU, bool F8, typename G>
__device__ __forceinline__ void f8_join(const F8GemmArgs& p, char* smem, const f32x16 (&acc)[G::FN][G::FM], int m0, int n0) {
  const int tid = threadIdx.x, lane = tid & 63, gw = tid >> 6;
  const int kg = gw / G::NW, wm = gw % G::NW / G::WN, wn = gw % G::WN;
  float* const parts = reinterpret_cast<float*>(smem);
  {
    float* const to = parts + (kg * G::BM + wm * G::WTM + (lane & 31)) * G::PITCH + wn * G::WTN + 4 * (lane >> 5);
#pragma unroll
    for (int i = 0; i < G::FN; ++i)
#pragma unroll
      for (int j = 0; j < G::FM; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<float4*>(to + 32 * j * G::PITCH + 32 * i + 8 * g) =
              make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
  }
  __syncthreads();
  constexpr int ES = F8 ? 1 : 2, PPR = G::BN / 8, NIT = (G::BM * PPR + G::THREADS - 1) / G::THREADS;
  static_assert(G::BM * PPR % 64 == 0 && (!F8 || PPR == 16), "whole waves of pieces");
  const int rows = min(G::BM, p.m - m0), cols = min(G::BN, p.n - n0);
  const F8Rows out{wave_rsrc(static_cast<char*>(p.c) + ((int64_t)m0 * p.ldc + n0) * ES, ((int64_t)(rows - 1) * p.ldc + cols) * ES),
                   (uint32_t)(p.ldc * ES), cols};
  const bool whole = (((uintptr_t)p.c & (8 * ES - 1)) | (p.ldc & 7) | (p.n & 7)) == 0;
#pragma unroll
  for (int it = 0; it < NIT; ++it) {
    const int pc = tid + it * G::THREADS, row = pc / PPR, col = pc % PPR * 8;
    if (pc >= G::BM * PPR) break;
    float v[8], o[8];
    Oct<float>::to(Oct<float>::load(parts + row * G::PITCH + col), v);
#pragma unroll
    for (int g = 1; g < G::KG; ++g) {
      Oct<float>::to(Oct<float>::load(parts + (g * G::BM + row) * G::PITCH + col), o);
#pragma unroll
      for (int r = 0; r < 8; ++r) v[r] += o[r];
    }
    Oct<T>::to(Oct<T>::load(reinterpret_cast<const T*>(smem + G::BIAS) + col), o);
#pragma unroll
    for (int r = 0; r < 8; ++r) v[r] += o[r];
    if constexpr (GELU && F8) {
      float top = 0.f, far = 0.f;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        o[r] = gelu_erf(v[r]);
        top = fmaxf(top, fabsf(o[r]));
        far = fmaxf(far, fabsf(v[r]));
      }
      // of the block (eight values alone are low often enough to cost 0.3 us)
      const bool low = gelu_is_low(row16_max(top), row16_max(far));
      if (__any(low)) {
#pragma unroll
        for (int r = 0; r < 8; ++r) o[r] = low ? gelu_low(v[r]) : o[r];
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) v[r] = o[r];
    } else if constexpr (GELU) {
#pragma unroll
      for (int r = 0; r < 8; ++r) v[r] = gelu_erf(v[r]);
    }
    if constexpr (F8) {
      float top = 0.f;  // N is a multiple of 4
#pragma unroll
      for (int r = 0; r < 8; ++r) top = fmaxf(top, col + (r & 4) < cols ? fabsf(v[r]) : 0.f);
      const float s = f8_scale(row16_max(top)), inv = __builtin_amdgcn_rcpf(s);
      const uint32_t x = f8_pack4(v[0], v[1], v[2], v[3], inv), y = f8_pack4(v[4], v[5], v[6], v[7], inv);
      if (col == 0 && row < rows) p.cs[(int64_t)(m0 + row) * p.ld_cs + n0 / 128] = s;
      if (whole) {
        out.put8(row, col, 1, x, y);
      } else {
        out.put4(row, col, 1, x);
        out.put4(row, col + 4, 1, y);
      }
    } else {
      const uint4 q = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
      if (whole) {
        out.put16<0>(row, col, 2, q);
      } else {
        out.put8(row, col, 2, q.x, q.y);
        out.put8(row, col + 4, 2, q.z, q.w);
      }
    }
  }
}

// Outputs in a 2-byte type T.  Lane (l32, hi) holds columns 32 i + 8 g + 4 hi
// .. + 3 of rows 32 j + l32: the lane halves trade quads, so that each holds whole
// 16-byte pieces, which go through `stage` (64 WTN bytes of the wave's own; piece c
// of row r at c ^ x(r), EpiStage's conflict-free order) to leave as row segments.
// All of a 32-row block's pieces are read before the first is stored.
template <typename T, typename G>
__device__ __forceinline__ void f8_store(const F8GemmArgs& p, const f32x16 (&acc)[G::FN][G::FM], int mw, int nw,
                                         int lane, char* stage) {
  typedef EpiStage<T, TJK_EPI_BIAS, G::FN> E;
  constexpr int LPR = E::LPR, NIT = 32 * LPR / 64;
  const int l32 = lane & 31, hi = lane >> 5;
  const F8Rows out = f8_rows<G>(p, mw, nw, 2);
  const bool whole = (((uintptr_t)p.c & 15) | (p.ldc & 7) | (p.n & 7)) == 0;
  const bool wt = (int64_t)p.m * p.n * 2 >= kWtMinBytes;
#pragma unroll
  for (int j = 0; j < G::FM; ++j) {
#pragma unroll
    for (int i = 0; i < G::FN; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const f32x16& a = acc[i][j];
        const int r = 8 * k;
        const auto s0 = __builtin_amdgcn_permlane32_swap(pack2<T>(a[r], a[r + 1]), pack2<T>(a[r + 4], a[r + 5]), false, false);
        const auto s1 = __builtin_amdgcn_permlane32_swap(pack2<T>(a[r + 2], a[r + 3]), pack2<T>(a[r + 6], a[r + 7]), false, false);
        *reinterpret_cast<uint4*>(stage + E::at(l32, 4 * i + 2 * k + hi)) = make_uint4(s0[0], s1[0], s0[1], s1[1]);
      }
    uint4 v[NIT];
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const int pc = lane + 64 * it;
      v[it] = *reinterpret_cast<const uint4*>(stage + E::at(pc / LPR, pc % LPR));
    }
    auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
      for (int it = 0; it < NIT; ++it) {
        const int pc = lane + 64 * it;
        f(32 * j + pc / LPR, pc % LPR * 8, v[it]);
      }
    };
    if (!whole) {
      each([&](int row, int col, const uint4& x) __attribute__((always_inline)) {
        out.put8(row, col, 2, x.x, x.y);
        out.put8(row, col + 4, 2, x.z, x.w);
      });
    } else if (wt) {
      each([&](int row, int col, const uint4& x) __attribute__((always_inline)) { out.put16<kStoreWt>(row, col, 2, x); });
    } else {
      each([&](int row, int col, const uint4& x) __attribute__((always_inline)) { out.put16<0>(row, col, 2, x); });
    }
  }
}

// Outputs in e4m3.  A row's largest magnitude over the wave's 64 columns takes
// one lane exchange; the two waves of a block of 128 trade theirs through LDS
// (`red`, BM x WN floats; every wave of the workgroup calls this).  Words are put in
// rows through `stage` (1024 FM FN bytes of the wave's own), the 16-byte piece c of row
// r at c ^ x(r).
template <typename G>
__device__ __forceinline__ void f8_quantise(const F8GemmArgs& p, const f32x16 (&acc)[G::FN][G::FM], int mw, int nw,
                                            int wm, int wn, int lane, float* red, char* stage) {
  constexpr int FM = G::FM, FN = G::FN;
  static_assert(FN == 2 && G::WN % 2 == 0, "two waves share a block, rows of 64 bytes");
  const int l32 = lane & 31, hi = lane >> 5;
  float top[FM];
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    top[j] = 0.f;
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float t = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) t = fmaxf(t, fabsf(acc[i][j][4 * g + r]));
        top[j] = fmaxf(top[j], nw + 32 * i + 8 * g + 4 * hi < p.n ? t : 0.f);
      }
    top[j] = fmaxf(top[j], __shfl_xor(top[j], 32));
  }
  if (hi == 0) {
#pragma unroll
    for (int j = 0; j < FM; ++j) red[wn * G::BM + wm * G::WTM + 32 * j + l32] = top[j];
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < FM; ++j)
    top[j] = fmaxf(top[j], red[(wn ^ 1) * G::BM + wm * G::WTM + 32 * j + l32]);
  constexpr int LPR = 4;  // pieces per row
  auto x = [](int r) { return (r >> 1) & 3; };
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const float s = f8_scale(top[j]), inv = __builtin_amdgcn_rcpf(s);
    const int m = mw + 32 * j + l32;
    if (hi == 0 && wn % 2 == 0 && m < p.m && nw < p.n) p.cs[(int64_t)m * p.ld_cs + nw / 128] = s;
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<uint32_t*>(stage + (32 * j + l32) * 16 * LPR + (((2 * i + (g >> 1)) ^ x(l32)) << 4) +
                                     8 * (g & 1) + 4 * hi) =
            f8_pack4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3], inv);
  }
  const F8Rows out = f8_rows<G>(p, mw, nw, 1);
  const bool whole = (((uintptr_t)p.c & 15) | (p.ldc & 15) | (p.n & 15)) == 0;
  const bool wt = (int64_t)p.m * p.n >= kWtMinBytes;
  constexpr int NIT = 32 * FM * LPR / 64;
  uint4 v[NIT];
#pragma unroll
  for (int it = 0; it < NIT; ++it) {
    const int pc = lane + 64 * it, r = pc / LPR;
    v[it] = *reinterpret_cast<const uint4*>(stage + r * 16 * LPR + ((pc % LPR ^ x(r & 31)) << 4));
  }
  auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const int pc = lane + 64 * it;
      f(pc / LPR, pc % LPR * 16, v[it]);
    }
  };
  if (!whole) {  // N and ldc are multiples of 4
    each([&](int row, int col, const uint4& q) __attribute__((always_inline)) {
      out.put4(row, col, 1, q.x);
      out.put4(row, col + 4, 1, q.y);
      out.put4(row, col + 8, 1, q.z);
      out.put4(row, col + 12, 1, q.w);
    });
  } else if (wt) {
    each([&](int row, int col, const uint4& q) __attribute__((always_inline)) { out.put16<kStoreWt>(row, col, 1, q); });
  } else {
    each([&](int row, int col, const uint4& q) __attribute__((always_inline)) { out.put16<0>(row, col, 1, q); });
  }
}

// Tile of workgroup `bid`: XCD-contiguous ranges of a raster in groups of about
// 1024 rows, so that the tiles that an XCD has at work at a time (one or two per CU)
// lie in a block near a square, whose operands take the least traffic into its L2.
template <int BM>
__device__ __forceinline__ void f8_tile_coords(int bid, int tiles_m, int tiles_n, int& pid_m, int& pid_n) {
  constexpr int ROWS = BM >= 256 ? 4 : BM >= 128 ? 8 : BM >= 64 ? 16 : 32;
  const int t = xcd_remap(bid, tiles_m * tiles_n), group = t / (ROWS * tiles_n);
  const int rows = min(tiles_m - group * ROWS, ROWS), in = t - group * (ROWS * tiles_n);
  if (rows == ROWS) {
    pid_m = group * ROWS + in % ROWS;
    pid_n = in / ROWS;
  } else {
    pid_m = group * ROWS + in % rows;
    pid_n = in / rows;
  }
}

// T: the bias's type, and the output's unless that is e4m3 (F8)
template <typename T, bool GELU, bool F8, typename G>
__global__ __launch_bounds__(G::THREADS, G::THREADS <= 256 && G::LDS > 80 * 1024 ? 1 : 2) void gemm_f8_kernel(F8GemmArgs p) {
  __shared__ __align__(16) char smem[G::LDS];
  int pid_m, pid_n;
  f8_tile_coords<G::BM>(blockIdx.x, (p.m + G::BM - 1) / G::BM, (p.n + G::BN - 1) / G::BN, pid_m, pid_n);
  const int m0 = pid_m * G::BM, n0 = pid_n * G::BN;
  const int gw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = gw % G::NW;
  // the bias of the tile's columns; zeros past N, and without one
  {
    const int lane = threadIdx.x & 63;
    const u32x4 r = lds_dma_rsrc(static_cast<const T*>(p.bias) + n0,
                                 p.bias != nullptr ? (int64_t)(p.n - n0) * (int64_t)sizeof(T) : 0);
    constexpr int NI = (G::BN * (int)sizeof(T) + 255) / 256;
    static_assert(NI * 256 <= G::BIAS_BYTES, "the DMA of the bias writes all of its words");
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (i % (G::NW * G::KG) == gw) {
        const int at = i * 256 + lane * 4;
        lds_dma4(r, at < G::BN * (int)sizeof(T) ? at : kPastEnd,
                 (uint32_t)(uintptr_t)(lds_void*)smem + G::BIAS + i * 256);
      }
  }
  f32x16 acc[G::FN][G::FM];
  zero_acc<float, G::FM, G::FN>(acc);
  f8_accumulate<G>(smem, p, m0, n0, acc);
  if constexpr (G::KG > 1) {
    f8_join<T, GELU, F8, G>(p, smem, acc, m0, n0);
    return;
  }
  // (an empty asm: nothing derived from the lane stays in a register through the main loop)
  int lane = threadIdx.x;
  asm volatile("" : "+v"(lane));
  lane &= 63;
  const int wm = wave / G::WN, wn = wave % G::WN;
  const int mw = m0 + wm * G::WTM, nw = n0 + wn * G::WTN;
  f8_values<T, GELU, F8, G>(smem, acc, wn, lane >> 5);
  if constexpr (F8) {
    constexpr int RED = G::BM * G::WN * 4;
    static_assert(RED + G::BM * G::BN <= G::BIAS, "epilogue staging");
    f8_quantise<G>(p, acc, mw, nw, wm, wn, lane, reinterpret_cast<float*>(smem), smem + RED + wave * 1024 * G::FM * G::FN);
  } else {
    static_assert(64 * G::WTN * G::NW <= G::BIAS, "epilogue staging");
    f8_store<T, G>(p, acc, mw, nw, lane, smem + wave * 64 * G::WTN);
  }
}

}  // namespace tjk

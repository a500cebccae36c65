// Entry point of the block-scaled e4m3 GEMM: argument checks and the choice
// of the tile.

#include "gemm_f8.h"

namespace tjk {

//             FM FN WM WN KG RA RW
typedef F8Geom<2, 4, 4, 2, 1, 4, 8, 9> Tile256;
typedef F8Geom<2, 4, 2, 2, 1, 3, 6> Tile128x256;
typedef F8Geom<3, 2, 2, 2, 1, 6, 4> Tile192x128;
typedef F8Geom<2, 2, 2, 2, 1, 4, 4> Tile128;
typedef F8Geom<1, 2, 2, 2, 1, 3, 6> Tile64x128;
typedef F8Geom<1, 2, 1, 1, 4, 2, 4> Tile32x64k4;
typedef F8Geom<1, 1, 1, 1, 4, 2, 2> Tile32k4;
typedef F8Geom<1, 1, 1, 1, 4, 4, 4> Tile32k4d;
typedef F8Geom<2, 2, 2, 4, 1, 4, 4> Tile128x256w8;
// of e4m3 outputs
typedef F8Geom<2, 2, 2, 2, 1, 4, 4, -1, true> Exact128;
typedef F8Geom<1, 2, 2, 2, 1, 3, 6, -1, true> Exact64x128;
typedef F8Geom<1, 2, 1, 2, 4, 3, 3, -1, true> Exact32x128k4;

template <typename T, bool GELU, bool F8, typename G>
static int run_tile(const F8GemmArgs& p, hipStream_t s) {
  const int64_t tiles = (int64_t)((p.m + G::BM - 1) / G::BM) * ((p.n + G::BN - 1) / G::BN);
  if (tiles * G::THREADS > UINT32_MAX) return fail(TJK_EUNSUPPORTED, "tjk_gemm_f8: %lld tiles are too many", (long long)tiles);
  gemm_f8_kernel<T, GELU, F8, G><<<(unsigned)tiles, G::THREADS, 0, s>>>(p);
  return check_launch("tjk_gemm_f8");
}

// Estimated microseconds of a launch on MI355X, as gemm.hip's estimate: with
// `tiles` workgroups, `per_cu` of them resident per CU, a launch is `rounds`
// fillings of the chip, in which the fullest CU runs `load` workgroups in all,
// each of `steps` K tiles (per K group), and stores `mb` MB of output:
//   c0 + c1 rounds + c2 rounds steps + c3 load + c4 load steps + c5 mb + c6 load (GELU)
// (mb at 5 TB/s).  Non-negative least squares, by relative error and weighted
// towards tiles near the best of their launch, over the 330 launches of
// profiles/gemm_f8_tiles.csv (1 to 16384 rows, widths and K from 128 to 8192, weights
// from memory), for e4m3 outputs over the 257 of profiles/gemm_f8_e4m3_tiles.csv.  The
// tile with the least estimate is 0.4% slower than the best of its list (e4m3: 0.2%,
// geometric means), none more than 9%, and of launches held out of the fit 0.5% (0.2%).
// Without one of the tiles the best would be slower by up to 2.0%; of the e4m3
// list by 3 to 4%, without 32 x 128 by 12%.
struct F8Plan {
  int bm, bn, per_cu, k_groups;
  float c[7];
};
static const F8Plan kPlans[] = {
    {Tile256::BM, Tile256::BN, 1, Tile256::KG, {1.392f, 3.643f, 0.000f, 0.000f, 1.448f, 0.706f, 5.415f}},
    {Tile128x256::BM, Tile128x256::BN, 2, Tile128x256::KG, {1.903f, 2.889f, 0.264f, 0.000f, 0.715f, 0.458f, 2.766f}},
    {Tile192x128::BM, Tile192x128::BN, 1, Tile192x128::KG, {1.204f, 3.131f, 0.000f, 0.000f, 0.737f, 0.360f, 2.286f}},
    {Tile128::BM, Tile128::BN, 2, Tile128::KG, {2.357f, 1.409f, 0.191f, 0.000f, 0.371f, 0.569f, 1.393f}},
    {Tile64x128::BM, Tile64x128::BN, 2, Tile64x128::KG, {3.136f, 0.289f, 0.213f, 0.000f, 0.219f, 1.188f, 0.683f}},
    {Tile32x64k4::BM, Tile32x64k4::BN, 1, Tile32x64k4::KG, {1.633f, 1.494f, 0.667f, 0.000f, 0.000f, 3.007f, 0.273f}},
    {Tile32k4::BM, Tile32k4::BN, 2, Tile32k4::KG, {2.107f, 0.750f, 0.489f, 0.000f, 0.153f, 4.449f, 0.221f}},
    {Tile32k4d::BM, Tile32k4d::BN, 1, Tile32k4d::KG, {1.910f, 0.000f, 0.512f, 1.250f, 0.000f, 5.385f, 0.260f}},
    {Tile128x256w8::BM, Tile128x256w8::BN, 1, Tile128x256w8::KG, {1.726f, 0.000f, 0.000f, 2.576f, 0.790f, 0.622f, 2.381f}}};
static const F8Plan kPlansF8[] = {
    {Exact128::BM, Exact128::BN, 2, Exact128::KG, {3.619f, 0.709f, 0.055f, 0.000f, 0.804f, 1.673f, 1.437f}},
    {Exact64x128::BM, Exact64x128::BN, 2, Exact64x128::KG, {3.735f, 0.335f, 0.168f, 0.000f, 0.438f, 2.554f, 0.665f}},
    {Exact32x128k4::BM, Exact32x128k4::BN, 1, Exact32x128k4::KG, {2.560f, 0.000f, 1.267f, 2.279f, 0.000f, 5.344f, 0.163f}}};
constexpr int kPlanCount = sizeof(kPlans) / sizeof(kPlans[0]), kPlanCountF8 = sizeof(kPlansF8) / sizeof(kPlansF8[0]);

// Rows are rounded up to a whole tile (256 at most) in 32-bit integers.
constexpr int64_t kMaxRows = (int64_t)INT32_MAX - 255;

// The tile with the least estimate.
static int auto_plan(int64_t m, int64_t n, int64_t k, bool f8, bool gelu) {
  int best = 0;
  float best_us = 0.f;
  for (int i = 0; i < (f8 ? kPlanCountF8 : kPlanCount); ++i) {
    const F8Plan& q = f8 ? kPlansF8[i] : kPlans[i];
    const int64_t tiles = ((m + q.bm - 1) / q.bm) * ((n + q.bn - 1) / q.bn), slots = 256 * q.per_cu;
    const int64_t full = tiles / slots, rest = tiles % slots;
    const float rounds = (float)(full + (rest > 0)), load = (float)(full * q.per_cu + (rest + 255) / 256);
    const float steps = (float)(((k + 127) / 128 + q.k_groups - 1) / q.k_groups);
    const float mb = (float)m * (float)n * (f8 ? 1.f : 2.f) / 5e6f;
    const float us = q.c[0] + rounds * (q.c[1] + q.c[2] * steps) + load * (q.c[3] + q.c[4] * steps) + q.c[5] * mb +
                     (gelu ? q.c[6] * load : 0.f);
    if (i == 0 || us < best_us) {
      best = i;
      best_us = us;
    }
  }
  return best;
}

template <typename T, bool GELU>
static int run_plan(int plan, const F8GemmArgs& p, hipStream_t s) {
  switch (plan) {
    case 0: return run_tile<T, GELU, false, Tile256>(p, s);
    case 1: return run_tile<T, GELU, false, Tile128x256>(p, s);
    case 2: return run_tile<T, GELU, false, Tile192x128>(p, s);
    case 3: return run_tile<T, GELU, false, Tile128>(p, s);
    case 4: return run_tile<T, GELU, false, Tile64x128>(p, s);
    case 5: return run_tile<T, GELU, false, Tile32x64k4>(p, s);
    case 6: return run_tile<T, GELU, false, Tile32k4>(p, s);
    case 7: return run_tile<T, GELU, false, Tile32k4d>(p, s);
    default: return run_tile<T, GELU, false, Tile128x256w8>(p, s);
  }
}

template <bool GELU>
static int run_plan_f8(int plan, const F8GemmArgs& p, hipStream_t s) {
  switch (plan) {
    case 0: return run_tile<float, GELU, true, Exact128>(p, s);
    case 1: return run_tile<float, GELU, true, Exact64x128>(p, s);
    default: return run_tile<float, GELU, true, Exact32x128k4>(p, s);
  }
}

}  // namespace tjk

using namespace tjk;

extern "C" int tjk_gemm_f8_plan_count(void) { return kPlanCount; }

extern "C" int tjk_gemm_f8_default_plan(int64_t m, int64_t n, int64_t k, int out_dtype, int epilogue) {
  if (m <= 0 || n <= 0 || k < 0 || m > kMaxRows || n > INT32_MAX || k > INT32_MAX)
    return fail(TJK_EINVAL, "tjk_gemm_f8_default_plan: bad shape");
  if (out_dtype != TJK_F16 && out_dtype != TJK_BF16 && out_dtype != TJK_E4M3)
    return fail(TJK_EINVAL, "tjk_gemm_f8_default_plan: bad output dtype %d", out_dtype);
  if (epilogue != TJK_EPI_BIAS && epilogue != TJK_EPI_BIAS_GELU)
    return fail(TJK_EINVAL, "tjk_gemm_f8_default_plan: bad epilogue %d", epilogue);
  return auto_plan(m, n, k, out_dtype == TJK_E4M3, epilogue == TJK_EPI_BIAS_GELU);
}

extern "C" int tjk_gemm_f8(const void* a, int64_t lda, const float* a_scales, int64_t ld_as, const void* w, int64_t ldw,
                           const float* w_scales, int64_t ld_ws, const void* bias, void* c, int out_dtype, int64_t ldc,
                           float* c_scales, int64_t ld_cs, int64_t m, int64_t n, int64_t k, int epilogue, int plan_id,
                           void* stream) {
  if (m < 0 || n < 0 || k < 0) return fail(TJK_EINVAL, "tjk_gemm_f8: negative shape");
  if (epilogue != TJK_EPI_BIAS && epilogue != TJK_EPI_BIAS_GELU)
    return fail(TJK_EINVAL, "tjk_gemm_f8: epilogue %d is neither the bias's nor GELU's", epilogue);
  if (out_dtype != TJK_F16 && out_dtype != TJK_BF16 && out_dtype != TJK_E4M3)
    return fail(TJK_EINVAL, "tjk_gemm_f8: output dtype %d is not a 2-byte one or e4m3", out_dtype);
  if (plan_id < -1 || plan_id >= kPlanCount)
    return fail(TJK_EINVAL, "tjk_gemm_f8: plan %d out of range [-1,%d)", plan_id, kPlanCount);
  if (m == 0 || n == 0) return TJK_OK;
  const bool f8 = out_dtype == TJK_E4M3;
  if (f8 && plan_id >= kPlanCountF8)
    return fail(TJK_EUNSUPPORTED, "tjk_gemm_f8: an e4m3 output has plans 0 to %d, not %d", kPlanCountF8 - 1, plan_id);
  if ((k && (!a || !w || !a_scales || !w_scales)) || !c || (f8 && !c_scales)) return fail(TJK_EINVAL, "tjk_gemm_f8: null pointer");
  if (m > INT32_MAX || n > INT32_MAX || k > INT32_MAX) return fail(TJK_EUNSUPPORTED, "tjk_gemm_f8: shape exceeds int32");
  if (m > kMaxRows) return fail(TJK_EUNSUPPORTED, "tjk_gemm_f8: %lld rows are too many", (long long)m);
  if (k % 16) return fail(TJK_EUNSUPPORTED, "tjk_gemm_f8: k=%lld must be a multiple of 16", (long long)k);
  if (n % 4) return fail(TJK_EUNSUPPORTED, "tjk_gemm_f8: n=%lld must be a multiple of 4", (long long)n);
  const int64_t kb = (k + kF8Block - 1) / kF8Block, nb = (n + kF8Block - 1) / kF8Block;
  if (lda < k || ldw < k || ldc < n || ld_as < kb || ld_ws < kb || (f8 && ld_cs < nb))
    return fail(TJK_EINVAL, "tjk_gemm_f8: leading dimension too small");
  if (lda % 16 || ldw % 16) return fail(TJK_EUNSUPPORTED, "tjk_gemm_f8: lda/ldw must be multiples of 16");
  if (ldc % 4) return fail(TJK_EUNSUPPORTED, "tjk_gemm_f8: ldc must be a multiple of 4");
  // 256 rows of an operand or of its scales, or 96 of the output (a wave's), within 31-bit
  // byte offsets; so n and k, at most ldc and lda, can be rounded up too
  if (ldc > INT32_MAX / 256 || lda > INT32_MAX / 256 || ldw > INT32_MAX / 256 || ld_as > INT32_MAX / 1024 || ld_ws > INT32_MAX / 1024)
    return fail(TJK_EUNSUPPORTED, "tjk_gemm_f8: leading dimension too large");
  const uintptr_t need_c = f8 ? 3 : 7, need_bias = f8 ? 15 : 7;
  if (((uintptr_t)a & 15) || ((uintptr_t)w & 15) || ((uintptr_t)c & need_c) || ((uintptr_t)bias & need_bias) ||
      ((uintptr_t)a_scales & 3) || ((uintptr_t)w_scales & 3) || ((uintptr_t)c_scales & 3))
    return fail(TJK_EUNSUPPORTED, "tjk_gemm_f8: misaligned pointer");
  const F8GemmArgs p{static_cast<const uint8_t*>(a), lda, a_scales, ld_as, static_cast<const uint8_t*>(w), ldw,
                     w_scales, ld_ws, bias, c, ldc, c_scales, ld_cs, (int)m, (int)n, (int)k};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool gelu = epilogue == TJK_EPI_BIAS_GELU;
  const int plan = plan_id >= 0 ? plan_id : auto_plan(m, n, k, f8, gelu);
  if (f8) return gelu ? run_plan_f8<true>(plan, p, s) : run_plan_f8<false>(plan, p, s);
  if (out_dtype == TJK_F16)
    return gelu ? run_plan<f16, true>(plan, p, s) : run_plan<f16, false>(plan, p, s);
  return gelu ? run_plan<bf16, true>(plan, p, s) : run_plan<bf16, false>(plan, p, s);
}

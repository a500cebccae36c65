// Entry point of the block-scaled e4m3 GEMM: argument checks and the choice
// of the tile.

#include "gemm_f8.h"

namespace tjk {

//             FM FN WM WN KG RA RW
typedef F8Geom<2, 4, 4, 2, 1, 4, 8, 9> Tile256;
typedef F8Geom<2, 4, 4, 2, 1, 4, 8> Tile256b;
typedef F8Geom<2, 4, 2, 2, 1, 3, 6> Tile128x256;
typedef F8Geom<2, 2, 2, 2, 1, 4, 4> Tile128;
typedef F8Geom<1, 2, 2, 2, 2, 3, 6> Tile64x128;

template <typename T, bool GELU, bool F8, typename G>
static int run_tile(const F8GemmArgs& p, hipStream_t s) {
  const int64_t tiles = (int64_t)((p.m + G::BM - 1) / G::BM) * ((p.n + G::BN - 1) / G::BN);
  if (tiles * G::THREADS > UINT32_MAX) return fail(TJK_EUNSUPPORTED, "tjk_gemm_f8: %lld tiles are too many", (long long)tiles);
  gemm_f8_kernel<T, GELU, F8, G><<<(unsigned)tiles, G::THREADS, 0, s>>>(p);
  return check_launch("tjk_gemm_f8");
}

struct F8Plan {
  int bm, bn, threads, k_groups;
};
#define TJK_F8_PLAN(G) {G::BM, G::BN, G::THREADS, G::KG}
static const F8Plan kPlans[] = {TJK_F8_PLAN(Tile256), TJK_F8_PLAN(Tile256b), TJK_F8_PLAN(Tile128x256), TJK_F8_PLAN(Tile128), TJK_F8_PLAN(Tile64x128)};
constexpr int kPlanCount = sizeof(kPlans) / sizeof(kPlans[0]);

template <typename T, bool GELU, bool F8>
static int run_plan(int plan, const F8GemmArgs& p, hipStream_t s) {
  switch (plan) {
    case 0: return run_tile<T, GELU, F8, Tile256>(p, s);
    case 1: return run_tile<T, GELU, F8, Tile256b>(p, s);
    case 2: return run_tile<T, GELU, F8, Tile128x256>(p, s);
    case 3: return run_tile<T, GELU, F8, Tile128>(p, s);
    default: return run_tile<T, GELU, F8, Tile64x128>(p, s);
  }
}

}  // namespace tjk

using namespace tjk;

extern "C" int tjk_gemm_f8_plan_count(void) { return kPlanCount; }

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
  if (!a || !w || !a_scales || !w_scales || !c || (f8 && !c_scales)) return fail(TJK_EINVAL, "tjk_gemm_f8: null pointer");
  if (m > INT32_MAX || n > INT32_MAX || k > INT32_MAX) return fail(TJK_EUNSUPPORTED, "tjk_gemm_f8: shape exceeds int32");
  if (k % 16) return fail(TJK_EUNSUPPORTED, "tjk_gemm_f8: k=%lld must be a multiple of 16", (long long)k);
  if (n % 4) return fail(TJK_EUNSUPPORTED, "tjk_gemm_f8: n=%lld must be a multiple of 4", (long long)n);
  const int64_t kb = (k + kF8Block - 1) / kF8Block, nb = (n + kF8Block - 1) / kF8Block;
  if (lda < k || ldw < k || ldc < n || ld_as < kb || ld_ws < kb || (f8 && ld_cs < nb))
    return fail(TJK_EINVAL, "tjk_gemm_f8: leading dimension too small");
  if (lda % 16 || ldw % 16) return fail(TJK_EUNSUPPORTED, "tjk_gemm_f8: lda/ldw must be multiples of 16");
  if (ldc % 4) return fail(TJK_EUNSUPPORTED, "tjk_gemm_f8: ldc must be a multiple of 4");
  // 256 rows of an operand, of its scales, or 64 of the output within 31-bit byte offsets
  if (ldc > INT32_MAX / 256 || lda > INT32_MAX / 256 || ldw > INT32_MAX / 256 || ld_as > INT32_MAX / 1024 || ld_ws > INT32_MAX / 1024)
    return fail(TJK_EUNSUPPORTED, "tjk_gemm_f8: leading dimension too large");
  const uintptr_t need_c = f8 ? 3 : 7, need_bias = f8 ? 15 : 7;
  if (((uintptr_t)a & 15) || ((uintptr_t)w & 15) || ((uintptr_t)c & need_c) || ((uintptr_t)bias & need_bias) ||
      ((uintptr_t)a_scales & 3) || ((uintptr_t)w_scales & 3) || ((uintptr_t)c_scales & 3))
    return fail(TJK_EUNSUPPORTED, "tjk_gemm_f8: misaligned pointer");
  const F8GemmArgs p{static_cast<const uint8_t*>(a), lda, a_scales, ld_as, static_cast<const uint8_t*>(w), ldw,
                     w_scales, ld_ws, bias, c, ldc, c_scales, ld_cs, (int)m, (int)n, (int)k};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int plan = plan_id >= 0 ? plan_id : 0;
  const bool gelu = epilogue == TJK_EPI_BIAS_GELU;
  if (f8) return gelu ? run_plan<float, true, true>(plan, p, s) : run_plan<float, false, true>(plan, p, s);
  if (out_dtype == TJK_F16)
    return gelu ? run_plan<f16, true, false>(plan, p, s) : run_plan<f16, false, false>(plan, p, s);
  return gelu ? run_plan<bf16, true, false>(plan, p, s) : run_plan<bf16, false, false>(plan, p, s);
}

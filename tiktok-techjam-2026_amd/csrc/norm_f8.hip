// Residual add + RMS norm with an output in e4m3 (or a wider type), and the
// quantisation of a matrix to e4m3 with block scales.

#include <type_traits>

#include "f8_common.h"

namespace tjk {

// ------------------------------------------------------------------ RMS norm
//
// x = res (+ delta), r = rsqrt(mean(x^2) + eps), y = x r gamma, all in fp32.
// A row belongs to T threads (whole waves); thread t holds the 8-element
// pieces t, t + T, ... in registers, so the row is read once.  A block of
// 128 columns is 16 neighbouring lanes, one DPP row: its largest magnitude
// needs no LDS.
//
// Bound by memory: residual, addend, sum and quantised row pass once, 7 bytes per
// element with 2-byte ones.  32768 x 4096 bf16: 165 us, 5.7 TB/s (a copy of 1 GB
// reaches 4.8; to bf16 186 us, to fp32 243); 5430 x 1024 with an fp32 residual: 11.3 us,
// 5.4 TB/s, as quick from one wave per row (four rows a workgroup) as it gets (to bf16
// 12.1).  1024 threads a row: 8192 x 16384 bf16 164 us, 5.7 TB/s; 4096 x 32768 190, 5.0.
// 8 x 2048: 2.6 us in a graph, a launch and two passages of memory latency.  gamma is
// loaded where it is used: requested with the row it takes registers, and 2 to 4% longer.

struct NormArgs {
  const void* res;
  int64_t ld_res;
  const void* delta;
  int64_t ld_delta;
  void* res_out;
  int ro_dtype;
  int64_t ld_ro;
  void* out;
  int out_dtype;
  int64_t ld_out;
  float* scales;
  int64_t ld_scales;
  const float* gamma;
  int64_t rows;
  int n;
  float eps;
};

// Piece p of a row in one of the three wide types.
__device__ __forceinline__ void put_piece(void* row, int dtype, int p, const float (&v)[8]) {
  if (dtype == TJK_F32) {
    static_cast<Oct<float>::raw*>(row)[p] = Oct<float>::from(v);
  } else if (dtype == TJK_F16) {
    static_cast<uint4*>(row)[p] = Oct<f16>::from(v);
  } else {
    static_cast<uint4*>(row)[p] = Oct<bf16>::from(v);
  }
}

template <typename TR, typename TD, int T, int MAXCH>
__global__ __launch_bounds__(T < 256 ? 256 : T) void add_rmsnorm_kernel(NormArgs a) {
  constexpr int NT = T < 256 ? 256 : T;
  constexpr int NW = T / 64;  // waves per row
  __shared__ float part[NT / 64];
  const int t = threadIdx.x % T;
  const int64_t row = (int64_t)blockIdx.x * (NT / T) + threadIdx.x / T;
  const bool live = row < a.rows;
  const int np = a.n >> 3;  // pieces of a row
  const int64_t src = live ? row : a.rows - 1;

  // Pieces past the row's end are read at its last piece and dropped: a load
  // under a lane's own condition would be waited for by itself.
  const TR* const res = static_cast<const TR*>(a.res) + src * a.ld_res;
  typename Oct<TR>::raw xr[MAXCH];
#pragma unroll
  for (int c = 0; c < MAXCH; ++c) xr[c] = Oct<TR>::load(res + 8 * min(t + c * T, np - 1));
  float x[MAXCH][8];
  if (a.delta != nullptr) {
    const TD* const delta = static_cast<const TD*>(a.delta) + src * a.ld_delta;
    typename Oct<TD>::raw dr[MAXCH];
#pragma unroll
    for (int c = 0; c < MAXCH; ++c) dr[c] = Oct<TD>::load(delta + 8 * min(t + c * T, np - 1));
#pragma unroll
    for (int c = 0; c < MAXCH; ++c) {
      float d[8];
      Oct<TR>::to(xr[c], x[c]);
      Oct<TD>::to(dr[c], d);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[c][i] += d[i];
    }
  } else {
#pragma unroll
    for (int c = 0; c < MAXCH; ++c) Oct<TR>::to(xr[c], x[c]);
  }

  float sum = 0.f;
#pragma unroll
  for (int c = 0; c < MAXCH; ++c) {
    if (t + c * T < np) {
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(x[c][i], x[c][i], sum);
    }
  }
  if (a.res_out != nullptr && live) {
    char* const ro = static_cast<char*>(a.res_out) + row * a.ld_ro * (a.ro_dtype == TJK_F32 ? 4 : 2);
#pragma unroll
    for (int c = 0; c < MAXCH; ++c)
      if (t + c * T < np) put_piece(ro, a.ro_dtype, t + c * T, x[c]);
  }
  sum = wave_sum(sum);
  if constexpr (NW > 1) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) sum += part[w];
  }
  if (!live) return;
  const float r = 1.0f / sqrtf(sum / (float)a.n + a.eps);

  char* const out = static_cast<char*>(a.out) + row * a.ld_out * (a.out_dtype == TJK_E4M3 ? 1 : a.out_dtype == TJK_F32 ? 4 : 2);
#pragma unroll
  for (int c = 0; c < MAXCH; ++c) {
    const int p = t + c * T;
    const bool in = p < np;
    float g[8];
    Oct<float>::to(Oct<float>::load(a.gamma + 8 * min(p, np - 1)), g);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[c][i] = x[c][i] * r * g[i];
    if (a.out_dtype == TJK_E4M3) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[c][i]));
      const float s = f8_scale(row16_max(in ? top : 0.f));
      const float inv = __builtin_amdgcn_rcpf(s);
      if (in) {
        reinterpret_cast<uint2*>(out)[p] = make_uint2(f8_pack4(x[c][0], x[c][1], x[c][2], x[c][3], inv),
                                                      f8_pack4(x[c][4], x[c][5], x[c][6], x[c][7], inv));
        if ((t & 15) == 0) a.scales[row * a.ld_scales + (p >> 4)] = s;
      }
    } else if (in) {
      put_piece(out, a.out_dtype, p, x[c]);
    }
  }
}

template <typename TR, typename TD>
static int launch_norm(const NormArgs& a, hipStream_t s) {
  // Threads per row: as few as hold the row in four pieces each.
  auto go = [&](auto tt, auto mc) {
    constexpr int T = decltype(tt)::value, MC = decltype(mc)::value, NT = T < 256 ? 256 : T;
    const int64_t per = NT / T;
    add_rmsnorm_kernel<TR, TD, T, MC><<<(unsigned)((a.rows + per - 1) / per), NT, 0, s>>>(a);
    return check_launch("tjk_add_rmsnorm");
  };
  std::integral_constant<int, 64> t64;
  std::integral_constant<int, 256> t256;
  std::integral_constant<int, 1024> t1024;
  std::integral_constant<int, 1> c1;
  std::integral_constant<int, 2> c2;
  std::integral_constant<int, 4> c4;
  if (a.n <= 512) return go(t64, c1);
  if (a.n <= 1024) return go(t64, c2);
  if (a.n <= 2048) return go(t256, c1);
  if (a.n <= 4096) return go(t256, c2);
  if (a.n <= 8192) return go(t256, c4);
  if (a.n <= 16384) return go(t1024, c2);
  return go(t1024, c4);
}

// -------------------------------------------------------------- quantisation
//
// Blocks of one row and 128 columns: 16 lanes hold a block, 8 elements each.
// The blocks of the matrix are numbered row by row; a wave takes kQuantBlocks of
// them, four at a time, so narrow rows share a wave and every load of the
// wave goes out before the first is used.  Bound by memory: 8192 x 8192 bf16 in
// 37.2 us, 5.5 TB/s.

constexpr int kQuantBlocks = 16;

template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, int64_t ld, uint8_t* __restrict__ q,
                                                            int64_t ld_q, float* __restrict__ scales, int64_t ld_s,
                                                            int64_t rows, int n, int nb) {
  constexpr int U = kQuantBlocks / 4;
  const int lane = threadIdx.x & 63, g = lane >> 4, l16 = lane & 15;
  const int64_t wave = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t first = wave * kQuantBlocks;
  const int64_t row0 = first / nb;
  const int b0 = (int)(first - row0 * nb);
  if (row0 >= rows) return;
  const float inv_nb = 1.0f / (float)nb;
  typename Oct<T>::raw raw[U];
  int64_t row[U];
  int blk[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    // block first + 4 u + g: b0 + 4 u + g < nb + 16, so the quotient below is
    // exact: it is at least 1 / (2 nb) away from a whole number
    const int b = b0 + 4 * u + g;
    const int over = (int)(((float)b + 0.5f) * inv_nb);
    row[u] = row0 + over;
    blk[u] = b - over * nb;
    const int64_t r = min(row[u], rows - 1);
    const int col = min(blk[u] * kF8Block + 8 * l16, n - 8);
    raw[u] = Oct<T>::load(x + r * ld + col);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float v[8];
    Oct<T>::to(raw[u], v);
    const int col = blk[u] * kF8Block + 8 * l16;
    const bool in = col < n && row[u] < rows;
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
    const float s = f8_scale(row16_max(in ? top : 0.f));
    const float inv = __builtin_amdgcn_rcpf(s);
    if (in) {
      *reinterpret_cast<uint2*>(q + row[u] * ld_q + col) =
          make_uint2(f8_pack4(v[0], v[1], v[2], v[3], inv), f8_pack4(v[4], v[5], v[6], v[7], inv));
      if (l16 == 0) scales[row[u] * ld_s + blk[u]] = s;
    }
  }
}

// Blocks of 128 rows and 128 columns: one workgroup holds a block in
// registers, 32 rows at a time over its 512 threads (4096 x 1024 fp32: 5.6 us,
// with 256 threads 6.1, with 1024 5.9).  2600 x 1008 fp32: a launch and one round
// of loads of 168 workgroups.  8192 x 8192 bf16: 37.1 us, 5.4 TB/s.
constexpr int kQuantThreads = 512;

template <typename T>
__global__ __launch_bounds__(kQuantThreads) void quantize_tiles_kernel(const T* __restrict__ x, int64_t ld,
                                                                       uint8_t* __restrict__ q, int64_t ld_q,
                                                                       float* __restrict__ scales, int64_t ld_s,
                                                                       int64_t rows, int n, int nb) {
  constexpr int STEP = kQuantThreads / 16, U = kF8Block / STEP;  // rows at a time, how often
  __shared__ float part[kQuantThreads / 64];
  const int t = threadIdx.x, l16 = t & 15;
  const int64_t rb = blockIdx.x / nb;
  const int cb = (int)(blockIdx.x - rb * nb);
  const int64_t r0 = rb * kF8Block + (t >> 4);
  const int col = cb * kF8Block + 8 * l16;
  typename Oct<T>::raw raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u) raw[u] = Oct<T>::load(x + min(r0 + STEP * u, rows - 1) * ld + min(col, n - 8));
  float top = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float v[8];
    Oct<T>::to(raw[u], v);
    // rows and columns past the end repeat values of this block, so they
    // leave its largest magnitude as it is
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
  }
  top = row16_max(top);
  top = fmaxf(top, __shfl_xor(top, 16));
  top = fmaxf(top, __shfl_xor(top, 32));
  if ((t & 63) == 0) part[t >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kQuantThreads / 64; ++w) top = fmaxf(top, part[w]);
  const float s = f8_scale(top);
  const float inv = __builtin_amdgcn_rcpf(s);
  if (t == 0) scales[rb * ld_s + cb] = s;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t r = r0 + STEP * u;
    if (r < rows && col < n) {
      float v[8];
      Oct<T>::to(raw[u], v);
      *reinterpret_cast<uint2*>(q + r * ld_q + col) =
          make_uint2(f8_pack4(v[0], v[1], v[2], v[3], inv), f8_pack4(v[4], v[5], v[6], v[7], inv));
    }
  }
}

template <typename T>
static int launch_quantize(const void* x, int64_t ld, void* q, int64_t ld_q, float* scales, int64_t ld_s, int64_t rows,
                           int64_t n, int block_rows, hipStream_t s) {
  const int64_t nb = (n + kF8Block - 1) / kF8Block;
  if (rows > ((int64_t)1 << 38)) return fail(TJK_EUNSUPPORTED, "tjk_quantize_f8: %lld rows are too many", (long long)rows);
  const int64_t blocks = (block_rows == 1 ? rows : (rows + kF8Block - 1) / kF8Block) * nb;
  const int64_t grid = block_rows == 1 ? (blocks + 4 * kQuantBlocks - 1) / (4 * kQuantBlocks) : blocks;
  if (grid > (int64_t)UINT32_MAX / kQuantThreads)
    return fail(TJK_EUNSUPPORTED, "tjk_quantize_f8: %lld blocks are too many", (long long)blocks);
  const T* xt = static_cast<const T*>(x);
  uint8_t* qt = static_cast<uint8_t*>(q);
  if (block_rows == 1)
    quantize_rows_kernel<T><<<(unsigned)grid, 256, 0, s>>>(xt, ld, qt, ld_q, scales, ld_s, rows, (int)n, (int)nb);
  else
    quantize_tiles_kernel<T><<<(unsigned)grid, kQuantThreads, 0, s>>>(xt, ld, qt, ld_q, scales, ld_s, rows, (int)n, (int)nb);
  return check_launch("tjk_quantize_f8");
}

static bool wide_type(int dt) { return dt == TJK_F32 || dt == TJK_F16 || dt == TJK_BF16; }
// Pieces are 8 elements: 8 bytes of e4m3, else 16 (fp32 pieces are two of 16).
static uintptr_t piece_mask(int dt) { return dt == TJK_E4M3 ? 7 : 15; }

}  // namespace tjk

using namespace tjk;

extern "C" int tjk_add_rmsnorm(const void* res, int res_dtype, int64_t ld_res, const void* delta, int delta_dtype,
                               int64_t ld_delta, void* res_out, int res_out_dtype, int64_t ld_res_out, void* out,
                               int out_dtype, int64_t ld_out, float* scales, int64_t ld_scales, const float* gamma,
                               int64_t rows, int64_t n, float eps, void* stream) {
  if (rows < 0 || n <= 0)
    return fail(TJK_EINVAL, "tjk_add_rmsnorm: bad shape rows=%lld n=%lld", (long long)rows, (long long)n);
  if (n % 8) return fail(TJK_EUNSUPPORTED, "tjk_add_rmsnorm: n=%lld not a multiple of 8", (long long)n);
  if (n > 32768) return fail(TJK_EUNSUPPORTED, "tjk_add_rmsnorm: n=%lld exceeds 32768", (long long)n);
  if (!wide_type(res_dtype) || (delta && !wide_type(delta_dtype)) || (res_out && !wide_type(res_out_dtype)) ||
      (out_dtype != TJK_E4M3 && !wide_type(out_dtype)))
    return fail(TJK_EINVAL, "tjk_add_rmsnorm: bad dtype (res %d, delta %d, res_out %d, out %d)", res_dtype, delta_dtype,
                res_out_dtype, out_dtype);
  if (rows == 0) return TJK_OK;
  if (!res || !out || !gamma || (out_dtype == TJK_E4M3 && !scales))
    return fail(TJK_EINVAL, "tjk_add_rmsnorm: null pointer");
  const int64_t nb = (n + kF8Block - 1) / kF8Block;
  if (ld_res < n || ld_out < n || (delta && ld_delta < n) || (res_out && ld_res_out < n) ||
      (out_dtype == TJK_E4M3 && ld_scales < nb))
    return fail(TJK_EINVAL, "tjk_add_rmsnorm: leading dimension too small");
  if (ld_res % 8 || ld_out % 8 || (delta && ld_delta % 8) || (res_out && ld_res_out % 8))
    return fail(TJK_EUNSUPPORTED, "tjk_add_rmsnorm: leading dimensions must be multiples of 8");
  if (((uintptr_t)res & 15) || ((uintptr_t)delta & 15) || ((uintptr_t)res_out & 15) ||
      ((uintptr_t)out & piece_mask(out_dtype)) || ((uintptr_t)gamma & 15) || ((uintptr_t)scales & 3))
    return fail(TJK_EUNSUPPORTED, "tjk_add_rmsnorm: misaligned pointer");
  // each thread writes the pieces that it has read, and no others' as long as
  // they lie in the same places
  if (res_out && ((res_out == res && (res_out_dtype != res_dtype || ld_res_out != ld_res)) ||
                  (res_out == delta && (res_out_dtype != delta_dtype || ld_res_out != ld_delta))))
    return fail(TJK_EINVAL, "tjk_add_rmsnorm: res_out may alias res or delta only in place (same dtype and leading "
                "dimension)");
  if (rows > INT32_MAX) return fail(TJK_EUNSUPPORTED, "tjk_add_rmsnorm: rows exceed int32");
  // the launch counts its threads in 32 bits
  if (rows > (int64_t)UINT32_MAX / (n <= 1024 ? 64 : n <= 8192 ? 256 : 1024) - 4)
    return fail(TJK_EUNSUPPORTED, "tjk_add_rmsnorm: %lld rows are too many", (long long)rows);
  const NormArgs a{res,    ld_res,    delta,  ld_delta,  res_out, res_out_dtype, ld_res_out, out,
                   out_dtype, ld_out, scales, ld_scales, gamma,   rows,          (int)n,     eps};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  auto with_delta = [&](auto tr) {
    typedef decltype(tr) TR;
    if (!delta || delta_dtype == TJK_BF16) return launch_norm<TR, bf16>(a, s);
    if (delta_dtype == TJK_F16) return launch_norm<TR, f16>(a, s);
    return launch_norm<TR, float>(a, s);
  };
  if (res_dtype == TJK_F32) return with_delta(0.0f);
  if (res_dtype == TJK_F16) return with_delta(f16(0));
  return with_delta(bf16(0));
}

extern "C" int tjk_quantize_f8(const void* x, int x_dtype, int64_t ld_x, void* q, int64_t ld_q, float* scales,
                               int64_t ld_scales, int64_t rows, int64_t n, int block_rows, void* stream) {
  if (rows < 0 || n <= 0)
    return fail(TJK_EINVAL, "tjk_quantize_f8: bad shape rows=%lld n=%lld", (long long)rows, (long long)n);
  if (block_rows != 1 && block_rows != kF8Block)
    return fail(TJK_EINVAL, "tjk_quantize_f8: block_rows=%d must be 1 or %d", block_rows, kF8Block);
  if (!wide_type(x_dtype)) return fail(TJK_EINVAL, "tjk_quantize_f8: bad dtype %d", x_dtype);
  if (n % 8) return fail(TJK_EUNSUPPORTED, "tjk_quantize_f8: n=%lld not a multiple of 8", (long long)n);
  if (n > (1 << 20)) return fail(TJK_EUNSUPPORTED, "tjk_quantize_f8: n=%lld exceeds 2^20", (long long)n);
  if (rows == 0) return TJK_OK;
  if (!x || !q || !scales) return fail(TJK_EINVAL, "tjk_quantize_f8: null pointer");
  if (ld_x < n || ld_q < n || ld_scales < (n + kF8Block - 1) / kF8Block)
    return fail(TJK_EINVAL, "tjk_quantize_f8: leading dimension too small");
  if (ld_x % 8 || ld_q % 8) return fail(TJK_EUNSUPPORTED, "tjk_quantize_f8: leading dimensions must be multiples of 8");
  if (((uintptr_t)x & 15) || ((uintptr_t)q & 7) || ((uintptr_t)scales & 3))
    return fail(TJK_EUNSUPPORTED, "tjk_quantize_f8: misaligned pointer");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (x_dtype == TJK_F32)
    return launch_quantize<float>(x, ld_x, q, ld_q, scales, ld_scales, rows, n, block_rows, s);
  if (x_dtype == TJK_F16) return launch_quantize<f16>(x, ld_x, q, ld_q, scales, ld_scales, rows, n, block_rows, s);
  return launch_quantize<bf16>(x, ld_x, q, ld_q, scales, ld_scales, rows, n, block_rows, s);
}

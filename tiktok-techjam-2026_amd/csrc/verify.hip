// Verification of drafted tokens against the target's probabilities.
//
// From node `cur` (at first the root) its children are tried in the order of
// their numbers.  p and q are the target's and the draft's distribution
// behind cur, and each child x was drawn from q.  After k refusals the
// residual distribution is r_k / W_k with
//     r_k = max(p - c_k q, 0),  W_k = sum r_k,  c_0 = 0, W_0 = 1, c_{k+1} = c_k + W_k:
// max(r_k / W_k - q, 0) is max(p - (c_k + W_k) q, 0) / W_k, as r_k > 0 where it is
// not zero.  A child is taken if u q(x) W_k < r_k(x); with none left the next
// token is drawn from r_k.  Products and sums in 64 bits: a decision at a border
// does not hang on the order of a sum.

#include <algorithm>

#include "tjk_common.h"

namespace tjk {

struct VerifyArgs {
  const float* target;
  const float* draft;
  int64_t ld_target, ld_draft;
  const int32_t* tokens;
  const int32_t* parents;
  const float* accept_u;
  const float* sample_u;
  const int32_t* cu_nodes;
  int32_t* path;
  int64_t ld_path;
  int32_t* count;
  int32_t* token;
  int* index_errors;
  struct Slot* slots;  // [batch][max_nodes][parts]
  int64_t rows;
  int batch, max_nodes, vocab;
  int parts, part;  // workgroups of a sequence, elements of each
  int polls;        // of a missing sum
};

// The walk needs p and q at the drafted tokens only, which the lanes of a wave
// gather at once, and a pass over the vocabulary for each refusal: the sum W_k.
// The last such sum also says where the next token lies, so that only the part
// that holds it is read again.  A sequence's vocabulary is cut into `parts`, a
// workgroup each; every one walks the same walk from the same numbers and meets
// the others at the sums only: each puts its own in the workspace and reads
// theirs.  It waits a bounded time: a sum that does not come (workgroups of other
// work may hold the chip) it computes itself, in the same order, so nothing hangs on
// who was there; a part that was missed once is looked for only once at the next
// sums, until it is there again.  Each of a sequence's sums has places of its own (a
// refusal takes one, and the end one: max_nodes at most), so that a workgroup that comes
// late finds all that the others left.
//
// 64 trees of up to 32 nodes over 128257 tokens: 36 to 38 us (one workgroup a sequence
// 77), of which the clearing of the sums' places 3 to 5; the distributions of the last
// nodes alone are 13 at a copy's rate, but a tree with five refusals makes five
// passes, one after the other, of about 5 us: 128 KB of p and as much of q by one CU,
// the waves' sums, and two passages of memory to the other parts and back.  A part's p and q held in registers
// for a second refusal at a node took 4 us off that, and added 0.6 to the 11 of four
// chains of six over 32000.

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kMostParts = 64;
// Workgroups of a launch: one per CU, so that they are all there, beside other work
// too.  64 trees over 128257: 37.7 us with 256, 34.8 with 512 (parts of 8192), 119 with
// 1024 (parts of 4096), which are not all there (298 while late ones did not find the
// sums that they had missed).
constexpr int kMostGroups = 256;
// Least elements of a part, us with 4096 / 8192 / 16384: chain over 32000 11.1 / 10.9 / 9.2 (no
// meeting), 16 trees over 50000 21.6 / 21.1 / 22.8, 4 over 128000 19.5 / 17.0 / 17.8, 64 over
// 10000 18.1 / 13.2 / 13.1, 4 chains over 32000 11.6 / 12.1 / 11.4, 64 12.6 / 14.2 / 14.0.
constexpr int kPartElements = 16384;
constexpr int kPolls = 256;  // of a missing sum: about 50 us

constexpr int kMostNodes = 64;

struct Slot {  // of a workgroup's sum: its halves, each with the number of the sum; zeros before
  uint64_t half[2];
};

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // rows may begin anywhere

// A draft's weight: none if it is negative or NaN, which could otherwise take a token
// that the target excludes.
__device__ __forceinline__ float drafted(float q) { return fmaxf(q, 0.f); }
__device__ __forceinline__ double residual(float p, double c, float q) {
  return fmax((double)p - c * (double)drafted(q), 0.);  // NaN: no weight
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

// Four weights from x on (WHOLE: all before `end`; else what there is).
template <bool WHOLE = false>
__device__ __forceinline__ void weights4(const float* p, const float* q, double c, int x, int end, double (&w)[4]) {
  float a[4] = {0, 0, 0, 0}, b[4] = {0, 0, 0, 0};
  if (WHOLE || x + 4 <= end) {
    const f32x4u v = *reinterpret_cast<const f32x4u*>(p + x);
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = v[i];
    if (c != 0) {
      const f32x4u u = *reinterpret_cast<const f32x4u*>(q + x);
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = u[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (x + i < end) a[i] = p[x + i], b[i] = c != 0 ? q[x + i] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = residual(a[i], c, b[i]);
}

__global__ __launch_bounds__(kThreads) void verify_kernel(VerifyArgs a) {
  __shared__ double wave_sums[2][kWaves], part_sums[kMostParts];
  __shared__ int missing;
  const int b = blockIdx.x % a.batch, part = blockIdx.x / a.batch;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t first = max(a.cu_nodes[b], 0);
  const int n = (int)min((int64_t)min(max(max(a.cu_nodes[b + 1], 0) - (int)first, 0), a.max_nodes), max(a.rows - first, (int64_t)0));
  int32_t* const path = a.path + b * a.ld_path;
  const bool writes = part == 0 && tid == 0;
  if (n == 0) {
    if (part == 0)
      for (int i = tid; i < a.max_nodes; i += kThreads) path[i] = -1;
    if (writes) a.count[b] = 0, a.token[b] = -1;
    return;
  }
  // lane j: node j, and p and q of its token behind its parent
  int parent = -1;
  float pj = 0.f, qj = 0.f, uj = 0.f;
  if (lane > 0 && lane < n) {
    parent = a.parents[first + lane];
    const int x = a.tokens[first + lane];
    uj = a.accept_u[first + lane];
    if (parent < 0 || parent >= lane) {
      parent = -1;
    } else if (x >= 0 && x < a.vocab) {
      pj = a.target[(first + parent) * a.ld_target + x];
      qj = drafted(a.draft[(first + parent) * a.ld_draft + x]);
    } else {
      pj = -1.f;  // of no token: refused
      if (part == 0 && wave == 0 && a.index_errors) atomicAdd(a.index_errors, 1);
    }
  }
  const float *p = a.target + first * a.ld_target, *q = a.draft + first * a.ld_draft;

  // A part's sum: its waves' stretches, each 256 elements at a time.
  int flip = 0;
  auto sum_part = [&](int which, double c) {
    const int lo = which * a.part + wave * (a.part / kWaves), end = min(min(lo + a.part / kWaves, (which + 1) * a.part), a.vocab);
    double s = 0;
    int x = lo + 4 * lane;
    for (; x - 4 * lane + 1024 <= end; x += 1024) {
      double w[4][4];
#pragma unroll
      for (int u = 0; u < 4; ++u) weights4<true>(p, q, c, x + 256 * u, end, w[u]);
#pragma unroll
      for (int u = 0; u < 4; ++u) s += (w[u][0] + w[u][1]) + (w[u][2] + w[u][3]);
    }
    for (; x < end; x += 256) {
      double w[4];
      weights4(p, q, c, x, end, w);
      s += (w[0] + w[1]) + (w[2] + w[3]);
    }
    s = wave_sum64(s);
    flip ^= 1;  // (the last sums may still be read)
    if (lane == 0) wave_sums[flip][wave] = s;
    __syncthreads();
    s = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s += wave_sums[flip][w];
    return s;
  };
  int round = 0;
  bool late = false;  // thread i < parts: part i's last sum did not come
  // The whole sum at (p, q, c); part_sums has the parts'.
  auto sum_all = [&](double c) {
    ++round;
    const double mine = sum_part(part, c);
    if (a.parts == 1) {
      if (tid == 0) part_sums[0] = mine;
      __syncthreads();
      return mine;
    }
    Slot* const slots = a.slots + ((int64_t)b * a.max_nodes + round - 1) * a.parts;
    const uint64_t bits = __builtin_bit_cast(uint64_t, mine), tag = (uint64_t)round << 32;
    if (tid == 0) {
      __hip_atomic_store(&slots[part].half[0], tag | (uint32_t)bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(&slots[part].half[1], tag | bits >> 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      missing = 0;
    }
    __syncthreads();
    if (tid < a.parts) {
      double sum = mine;
      if (tid != part) {
        uint64_t lo = 0, hi = 0;
        bool there = false;
        const int polls = late ? min(a.polls, 1) : a.polls;
        for (int i = 0; i < polls && !there; ++i) {
          if (i > 0) __builtin_amdgcn_s_sleep(1);
          lo = __hip_atomic_load(&slots[tid].half[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          hi = __hip_atomic_load(&slots[tid].half[1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          there = lo >> 32 == (uint64_t)round && hi >> 32 == (uint64_t)round;
        }
        late = !there;
        sum = there ? __builtin_bit_cast(double, hi << 32 | (uint32_t)lo) : -1;
        if (late) missing = 1;
      }
      part_sums[tid] = sum;
    }
    __syncthreads();
    if (missing) {
      for (int i = 0; i < a.parts; ++i) {
        if (part_sums[i] >= 0) continue;  // (the same in every thread)
        const double s = sum_part(i, c);
        __syncthreads();
        if (tid == 0) part_sums[i] = s;
        __syncthreads();
      }
      sum_part(part, c);  // its waves' sums again, which the search wants
    }
    double s = 0;
    for (int i = 0; i < a.parts; ++i) s += part_sums[i];
    return s;
  };

  int cur = 0, done = 1, tried = 0;
  if (writes) path[0] = 0;
  double c = 0, mass = 1;
  bool summed = false;  // mass is the sum at c
  while (true) {
    const uint64_t left = __ballot(parent == cur && lane > tried);
    if (left == 0) break;
    const int j = __ffsll((unsigned long long)left) - 1;
    tried = j;
    const float pt = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, pj), j));
    const float qt = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, qj), j));
    const float ut = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, uj), j));
    if ((double)ut * (double)qt * mass < residual(pt, c, c == 0 ? 0.f : qt)) {
      if (writes) path[done] = j;
      ++done;
      cur = j;
      c = 0;
      mass = 1;
      summed = false;
      p = a.target + (first + j) * a.ld_target;
      q = a.draft + (first + j) * a.ld_draft;
    } else {
      c += mass;
      mass = sum_all(c);
      summed = true;
    }
  }
  if (part == 0)
    for (int i = done + tid; i < a.max_nodes; i += kThreads) path[i] = -1;
  if (!summed) mass = sum_all(c);
  if (!(mass > 0) && c != 0) {
    c = 0;
    mass = sum_all(c);
  }
  if (writes) a.count[b] = done;
  if (!(mass > 0)) {
    if (writes) a.token[b] = -1;
    return;
  }
  // the part, and in it the wave, whose sum passes the point; if rounding leaves
  // none, the last with any weight
  const double point = (double)a.sample_u[b] * mass;
  double before = 0, cum = 0;
  int where = -1;
  for (int i = 0; i < a.parts; ++i) {
    if (part_sums[i] > 0) where = i, before = cum;
    cum += part_sums[i];
    if (cum > point && part_sums[i] > 0) break;
  }
  if (where != part) return;
  cum = before;
  int at = 0;
  for (int w = 0; w < kWaves; ++w) {
    const double s = wave_sums[flip][w];
    if (s > 0) at = w, before = cum;
    cum += s;
    if (cum > point && s > 0) break;
  }
  if (at != wave) return;
  // 1024 elements at a time, 16 to a lane
  const int lo = part * a.part + wave * (a.part / kWaves), end = min(min(lo + a.part / kWaves, (part + 1) * a.part), a.vocab);
  int last = -1;
  for (int x0 = lo; x0 < end; x0 += 1024) {
    const int x = x0 + 16 * lane;
    double w[4][4], s = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) weights4(p, q, c, x + 4 * u, end, w[u]);
    int mine = -1;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s += w[i >> 2][i & 3];
      if (w[i >> 2][i & 3] > 0) mine = x + i;
    }
    double incl = s;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double up = __shfl_up(incl, d);
      if (lane >= d) incl += up;
    }
    const uint64_t some = __ballot(mine >= 0), past = __ballot(before + incl > point && s > 0);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      if (lane == l) {
        double run = before + incl - s;
        int token = mine;
#pragma unroll
        for (int i = 15; i >= 0; --i) {
          double upto = run;
#pragma unroll
          for (int k = 0; k <= i; ++k) upto += w[k >> 2][k & 3];
          if (upto > point && w[i >> 2][i & 3] > 0) token = x + i;
        }
        a.token[b] = token;
      }
      return;
    }
    if (some) last = __builtin_amdgcn_readlane(mine, 63 - __builtin_clzll(some));
    before += __shfl(incl, 63);
  }
  if (lane == 0) a.token[b] = last;
}

__global__ __launch_bounds__(256) void clear_slots_kernel(Slot* p, int n) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) *reinterpret_cast<uint4*>(p + i) = make_uint4(0, 0, 0, 0);
}

// Workgroups of a sequence.
static int verify_parts(int64_t vocab, int batch) {
  const int64_t most = std::min<int64_t>(kMostParts, batch > 0 ? kMostGroups / batch : 1);
  return (int)std::max<int64_t>(1, std::min(most, vocab / kPartElements));
}

}  // namespace tjk

using namespace tjk;

extern "C" size_t tjk_verify_tree_bytes(int64_t vocab, int batch) {
  if (vocab <= 0 || vocab > 1 << 24 || batch <= 0 || batch > 1 << 20) return 0;
  const int parts = verify_parts(vocab, batch);
  return parts > 1 ? (size_t)batch * kMostNodes * parts * sizeof(Slot) : 0;
}

static int verify_tree(const float* target, int64_t ld_target, const float* draft, int64_t ld_draft,
                       const int32_t* tokens, const int32_t* parents, const float* accept_u, const float* sample_u,
                       const int32_t* cu_nodes, int32_t* path, int64_t ld_path, int32_t* count, int32_t* token,
                       int* index_errors, int64_t rows, int64_t vocab, int batch, int max_nodes, void* workspace,
                       size_t workspace_bytes, int polls, void* stream) {
  const char* const who = "tjk_verify_tree";
  if (rows < 0 || vocab <= 0 || batch < 0 || max_nodes <= 0)
    return fail(TJK_EINVAL, "%s: bad shape rows=%lld vocab=%lld batch=%d max_nodes=%d", who, (long long)rows,
                (long long)vocab, batch, max_nodes);
  if (max_nodes > kMostNodes) return fail(TJK_EUNSUPPORTED, "%s: max_nodes=%d exceeds 64", who, max_nodes);
  if (rows > INT32_MAX || vocab > 1 << 24 || batch > 1 << 20) return fail(TJK_EUNSUPPORTED, "%s: too large", who);
  if (batch == 0) return TJK_OK;
  if (!cu_nodes || !path || !count || !token || !sample_u ||
      (rows > 0 && (!target || !draft || !tokens || !parents || !accept_u)))
    return fail(TJK_EINVAL, "%s: null pointer", who);
  if (ld_target < vocab || ld_draft < vocab || ld_path < max_nodes)
    return fail(TJK_EINVAL, "%s: leading dimension too small", who);
  const size_t need = tjk_verify_tree_bytes(vocab, batch);
  if (workspace_bytes < need || (need > 0 && !workspace))
    return fail(TJK_EINVAL, "%s: a workspace of %zu bytes, %zu needed", who, workspace ? workspace_bytes : 0, need);
  if ((uintptr_t)workspace & 15) return fail(TJK_EUNSUPPORTED, "%s: misaligned workspace", who);
  const int parts = verify_parts(vocab, batch);
  const int64_t part = ((vocab + parts - 1) / parts + 256 * kWaves - 1) / (256 * kWaves) * (256 * kWaves);
  const VerifyArgs a{target, draft, ld_target, ld_draft, tokens, parents, accept_u, sample_u, cu_nodes, path, ld_path, count,
                     token, index_errors, static_cast<Slot*>(workspace), rows, batch, max_nodes, (int)vocab, parts, (int)part, polls};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (parts > 1) {
    const int slots = batch * max_nodes * parts;
    clear_slots_kernel<<<(unsigned)((slots + 255) / 256), 256, 0, s>>>(a.slots, slots);
    if (const int bad = check_launch(who)) return bad;
  }
  verify_kernel<<<(unsigned)(batch * parts), kThreads, 0, s>>>(a);
  return check_launch(who);
}

extern "C" int tjk_verify_tree(const float* target, int64_t ld_target, const float* draft, int64_t ld_draft,
                               const int32_t* tokens, const int32_t* parents, const float* accept_u, const float* sample_u,
                               const int32_t* cu_nodes, int32_t* path, int64_t ld_path, int32_t* count, int32_t* token,
                               int* index_errors, int64_t rows, int64_t vocab, int batch, int max_nodes, void* workspace,
                               size_t workspace_bytes, void* stream) {
  return verify_tree(target, ld_target, draft, ld_draft, tokens, parents, accept_u, sample_u, cu_nodes, path, ld_path, count,
                     token, index_errors, rows, vocab, batch, max_nodes, workspace, workspace_bytes, kPolls, stream);
}

// The same for tests, with the looks at a missing sum given: with none every workgroup
// computes every sum itself.
extern "C" int tjk_verify_tree_polls(const float* target, int64_t ld_target, const float* draft, int64_t ld_draft,
                                     const int32_t* tokens, const int32_t* parents, const float* accept_u,
                                     const float* sample_u, const int32_t* cu_nodes, int32_t* path, int64_t ld_path,
                                     int32_t* count, int32_t* token, int* index_errors, int64_t rows, int64_t vocab, int batch,
                                     int max_nodes, void* workspace, size_t workspace_bytes, int polls, void* stream) {
  return verify_tree(target, ld_target, draft, ld_draft, tokens, parents, accept_u, sample_u, cu_nodes, path, ld_path, count,
                     token, index_errors, rows, vocab, batch, max_nodes, workspace, workspace_bytes, polls, stream);
}

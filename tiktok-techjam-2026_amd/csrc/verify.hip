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
  int64_t rows;
  int max_nodes, vocab;
};

constexpr int kVerifyThreads = 1024;

__device__ __forceinline__ double residual(float p, double c, float q) {
  const double r = (double)p - c * (double)q;
  return r > 0 ? r : 0;  // NaN: no weight
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

__global__ __launch_bounds__(kVerifyThreads) void verify_kernel(VerifyArgs a) {
  constexpr int NW = kVerifyThreads / 64;
  __shared__ double part[NW];
  __shared__ int found[NW];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t first = max(a.cu_nodes[b], 0);
  const int n = (int)min((int64_t)min(max(a.cu_nodes[b + 1] - a.cu_nodes[b], 0), a.max_nodes), max(a.rows - first, (int64_t)0));
  const int parent = lane > 0 && lane < n ? a.parents[first + lane] : -1;
  int32_t* const path = a.path + b * a.ld_path;
  if (n == 0) {
    for (int i = tid; i < a.max_nodes; i += kVerifyThreads) path[i] = -1;
    if (tid == 0) a.count[b] = 0, a.token[b] = -1;
    return;
  }
  // a thread's elements lie together, so the threads' sums are in order
  const int per = (a.vocab + kVerifyThreads - 1) / kVerifyThreads;
  const int lo = min(tid * per, a.vocab), hi = min(lo + per, a.vocab);
  auto thread_sum = [&](const float* p, const float* q, double c) {
    double s = 0;
    for (int x = lo; x < hi; ++x) s += residual(p[x], c, c == 0 ? 0.f : q[x]);
    return s;
  };
  auto block_sum = [&](double s) {
    s = wave_sum64(s);
    __syncthreads();
    if (lane == 0) part[wave] = s;
    __syncthreads();
    s = 0;
    for (int w = 0; w < NW; ++w) s += part[w];
    return s;
  };
  int cur = 0, done = 1, tried = 0;
  if (tid == 0) path[0] = 0;
  double c = 0, mass = 1;
  const float *p = a.target + first * a.ld_target, *q = a.draft + first * a.ld_draft;
  while (true) {
    const uint64_t left = __ballot(parent == cur && lane > tried);
    if (left == 0) break;
    const int j = __ffsll((unsigned long long)left) - 1;
    tried = j;
    const int x = a.tokens[first + j];
    bool taken = false;
    if (x >= 0 && x < a.vocab)
      taken = (double)a.accept_u[first + j] * (double)q[x] * mass < residual(p[x], c, c == 0 ? 0.f : q[x]);
    else if (tid == 0 && a.index_errors)
      atomicAdd(a.index_errors, 1);
    if (taken) {
      if (tid == 0) path[done] = j;
      ++done;
      cur = j;
      c = 0;
      mass = 1;
      p = a.target + (first + j) * a.ld_target;
      q = a.draft + (first + j) * a.ld_draft;
    } else {
      c += mass;
      mass = block_sum(thread_sum(p, q, c));
    }
  }
  for (int i = done + tid; i < a.max_nodes; i += kVerifyThreads) path[i] = -1;
  double mine = thread_sum(p, q, c), sum = block_sum(mine);
  if (!(sum > 0)) {
    c = 0;
    mine = thread_sum(p, q, c);
    sum = block_sum(mine);
  }
  // running sums: of the waves before, of the lanes before
  double before = 0;
  for (int w = 0; w < wave; ++w) before += part[w];
  double incl = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double up = __shfl_up(incl, d);
    if (lane >= d) incl += up;
  }
  double at = before + incl - mine;
  const double point = (double)a.sample_u[b] * sum;
  int mine_first = INT32_MAX, last = -1;
  for (int x = lo; x < hi; ++x) {
    const double r = residual(p[x], c, c == 0 ? 0.f : q[x]);
    at += r;
    if (r > 0) last = x;
    if (at > point && r > 0) {
      mine_first = x;
      break;
    }
  }
  // the first token past the point; if rounding leaves none, the last with any weight
  for (int d = 1; d < 64; d <<= 1) {
    mine_first = min(mine_first, __shfl_xor(mine_first, d));
    last = max(last, __shfl_xor(last, d));
  }
  __shared__ int lasts[NW];
  if (lane == 0) found[wave] = mine_first, lasts[wave] = last;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < NW; ++w) mine_first = min(mine_first, found[w]), last = max(last, lasts[w]);
    a.count[b] = done;
    a.token[b] = mine_first != INT32_MAX ? mine_first : last;
  }
}

}  // namespace tjk

using namespace tjk;

extern "C" int tjk_verify_tree(const float* target, int64_t ld_target, const float* draft, int64_t ld_draft,
                               const int32_t* tokens, const int32_t* parents, const float* accept_u, const float* sample_u,
                               const int32_t* cu_nodes, int32_t* path, int64_t ld_path, int32_t* count, int32_t* token,
                               int* index_errors, int64_t rows, int64_t vocab, int batch, int max_nodes, void* stream) {
  const char* const who = "tjk_verify_tree";
  if (rows < 0 || vocab <= 0 || batch < 0 || max_nodes <= 0)
    return fail(TJK_EINVAL, "%s: bad shape rows=%lld vocab=%lld batch=%d max_nodes=%d", who, (long long)rows,
                (long long)vocab, batch, max_nodes);
  if (max_nodes > 64) return fail(TJK_EUNSUPPORTED, "%s: max_nodes=%d exceeds 64", who, max_nodes);
  if (rows > INT32_MAX || vocab > 1 << 24 || batch > 1 << 20) return fail(TJK_EUNSUPPORTED, "%s: too large", who);
  if (batch == 0) return TJK_OK;
  if (!cu_nodes || !path || !count || !token || !sample_u ||
      (rows > 0 && (!target || !draft || !tokens || !parents || !accept_u)))
    return fail(TJK_EINVAL, "%s: null pointer", who);
  if (ld_target < vocab || ld_draft < vocab || ld_path < max_nodes)
    return fail(TJK_EINVAL, "%s: leading dimension too small", who);
  const VerifyArgs a{target, draft, ld_target, ld_draft, tokens, parents, accept_u, sample_u, cu_nodes, path, ld_path, count,
                     token, index_errors, rows, max_nodes, (int)vocab};
  verify_kernel<<<(unsigned)batch, kVerifyThreads, 0, reinterpret_cast<hipStream_t>(stream)>>>(a);
  return check_launch(who);
}

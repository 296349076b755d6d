// Verification of drafted tokens for gfx950: which of a sequence's drafts are
// kept, and the token drawn after them, from given random numbers.
//
//   draft i is kept while u_i q_i(x_i) < p_i(x_i)   (exact: products of two
//   24-bit significands in 64 bits)
//   weights w(v) = max(p_j(v) - q_j(v), 0) at the first draft j that is not, p_j
//   after all of them; the token is the lowest v with sum_{i<=v} w(i) > u W
//
// Sums are in 64 bits: in 32 a vocabulary's running sum is off by more than a
// rare token's probability.
#include "internal.h"

namespace oxi {
namespace {

constexpr int NT = 1024;

struct VerifyArgs {
  const float* target;
  const float* draft;
  const int64_t* tokens;
  const int64_t* lengths;
  const float* uniforms;
  int64_t* accepted;
  int64_t* out;
  int64_t batch, drafts, vocab;
  int* guard;
};

// How many drafts of the sequence are kept, to every thread of the block;
// `slot`: one int64 of LDS. `rejected`: whether a draft was not.
template <int N>
__device__ __forceinline__ int64_t count_kept(const VerifyArgs& g, int64_t b, unsigned long long* slot,
                                              bool& rejected) {
  int64_t len = g.lengths ? g.lengths[b] : g.drafts;
  const bool bad_len = len < 0 || len > g.drafts;
  len = min(max(len, (int64_t)0), g.drafts);
  if (threadIdx.x == 0) {
    *slot = (unsigned long long)len;
    if (bad_len) atomicOr(g.guard, 1);
  }
  __syncthreads();
  for (int64_t i = threadIdx.x; i < len; i += N) {
    const int64_t x = g.tokens[b * g.drafts + i];
    bool kept = false;
    if (x < 0 || x >= g.vocab) {
      atomicOr(g.guard, 1);
    } else {
      const double p = g.target[(b * (g.drafts + 1) + i) * g.vocab + x];
      const double q = g.draft ? (double)g.draft[(b * g.drafts + i) * g.vocab + x] : 1.0;
      kept = (double)g.uniforms[b * (g.drafts + 1) + i] * q < p;
    }
    if (!kept) atomicMin(slot, (unsigned long long)i);
  }
  __syncthreads();
  const int64_t kept = (int64_t)*slot;
  rejected = kept < len;
  return kept;
}

// The weights of a row: those left by the draft, and the target's own.
struct Row {
  const float* p;
  const float* q;   // NULL: nothing to take away
  int64_t removed;  // a class without weight (drafts without probabilities), or -1
  __device__ __forceinline__ double own(int64_t v) const { return p[v] > 0.f ? (double)p[v] : 0.0; }
  __device__ __forceinline__ double left(int64_t v) const {
    if (v == removed) return 0.0;
    if (!q) return own(v);
    const double d = (double)p[v] - (double)q[v];
    return d > 0.0 ? d : 0.0;
  }
};

__device__ __forceinline__ Row row_of(const VerifyArgs& g, int64_t b, int64_t kept, bool rejected) {
  Row r;
  r.p = g.target + (b * (g.drafts + 1) + kept) * g.vocab;
  r.q = rejected && g.draft ? g.draft + (b * g.drafts + kept) * g.vocab : nullptr;
  r.removed = rejected && !g.draft ? g.tokens[b * g.drafts + kept] : -1;
  return r;
}

template <int N>
__device__ __forceinline__ double block_sum(double v, double* lds) {
  v = wave_sum<double>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = lds[0];
#pragma unroll
  for (int i = 1; i < N / 64; ++i) s += lds[i];
  return s;
}

// Sum over the threads before this one, in order; `all` gets the whole sum.
template <int N>
__device__ __forceinline__ double block_before(double v, double* lds, double& all) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  double s = v;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const double o = __shfl_up(s, m, 64);
    if (lane >= m) s += o;
  }
  __syncthreads();
  if (lane == 63) lds[wid] = s;
  __syncthreads();
  double base = 0.0;
  all = 0.0;
#pragma unroll
  for (int i = 0; i < N / 64; ++i) {
    if (i < wid) base += lds[i];
    all += lds[i];
  }
  return base + (s - v);
}

// A block a sequence.
__global__ __launch_bounds__(NT) void verify_k(const VerifyArgs g) {
  __shared__ unsigned long long slot, found;
  __shared__ double red[NT / 64];
  __shared__ long long last;
  const int64_t b = blockIdx.x;
  const int t = threadIdx.x;
  bool rejected;
  const int64_t kept = count_kept<NT>(g, b, &slot, rejected);
  const Row r = row_of(g, b, kept, rejected);
  double own = 0.0, left = 0.0;
  for (int64_t v = t; v < g.vocab; v += NT) {
    own += r.own(v);
    left += r.left(v);
  }
  own = block_sum<NT>(own, red);
  left = block_sum<NT>(left, red);
  const bool use_left = rejected && left > 0.0;
  const double limit = (double)g.uniforms[b * (g.drafts + 1) + g.drafts] * (use_left ? left : own);
  if (t == 0) {
    found = ~0ull;
    last = -1;
  }
  __syncthreads();
  double carry = 0.0;
  for (int64_t v0 = 0; v0 < g.vocab; v0 += NT) {
    const int64_t v = v0 + t;
    const double w = v < g.vocab ? (use_left ? r.left(v) : r.own(v)) : 0.0;
    double all;
    const double before = carry + block_before<NT>(w, red, all);
    if (w > 0.0) {
      if (before + w > limit) atomicMin(&found, (unsigned long long)v);
      atomicMax(&last, (long long)v);
    }
    carry += all;
    __syncthreads();
    if (found != ~0ull) break;
  }
  const int64_t token = found != ~0ull ? (int64_t)found : last;
  if (t == 0) g.accepted[b] = kept;
  for (int64_t i = t; i <= g.drafts; i += NT)
    g.out[b * (g.drafts + 1) + i] = i < kept ? g.tokens[b * g.drafts + i] : i == kept ? token : -1;
}

}  // namespace
}  // namespace oxi

using namespace oxi;

extern "C" {

int oxi_verify_drafts_workspace(int64_t batch, int64_t vocab, int64_t* bytes) {
  if (batch < 0 || vocab < 0) return fail(OXI_INVALID_ARGUMENT, "verify_drafts_workspace: negative size");
  if (!bytes) return fail(OXI_INVALID_ARGUMENT, "verify_drafts_workspace: NULL result pointer");
  *bytes = 0;
  return OXI_OK;
}

int oxi_verify_drafts(const float* target, const float* draft, const int64_t* tokens, const int64_t* lengths,
                      const float* uniforms, int64_t* accepted, int64_t* out, void* workspace, int64_t batch,
                      int64_t drafts, int64_t vocab) {
  if (batch < 0 || drafts < 0 || vocab < 0) return fail(OXI_INVALID_ARGUMENT, "verify_drafts: negative size");
  if (vocab > ((int64_t)1 << 30) || batch > ((int64_t)1 << 20) || drafts > ((int64_t)1 << 20))
    return fail(OXI_INVALID_ARGUMENT, "verify_drafts: size exceeds the kernel limits");
  if (batch == 0) return OXI_OK;
  if (vocab == 0) return fail(OXI_INVALID_ARGUMENT, "verify_drafts: zero classes");
  if (!target || (drafts && !tokens) || !uniforms || !accepted || !out)
    return fail(OXI_INVALID_ARGUMENT, "verify_drafts: NULL tensor pointer");
  if (reinterpret_cast<uintptr_t>(workspace) & 7u)
    return fail(OXI_INVALID_ARGUMENT, "verify_drafts: the workspace at %p is not 8-byte aligned", workspace);
  OXI_CHECK_INIT();
  const VerifyArgs g{target, draft, tokens, lengths, uniforms, accepted, out, batch, drafts, vocab, guard_flag()};
  verify_k<<<dim3((unsigned)batch), dim3(NT), 0, stream()>>>(g);
  return check_launch("verify_drafts");
}

}  // extern "C"

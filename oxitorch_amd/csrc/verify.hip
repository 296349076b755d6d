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
#include "rowtile.h"

namespace oxi {
namespace {

constexpr int NT = 256;

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

// ---------------------------------------------------------------------------
// Two launches: the first cuts each sequence's row into chunks of NT threads x
// U float4s, a block a chunk, which sums its weights; the second, a block a
// sequence, finds the chunk that the drawn number falls into and reads that
// one again. Each block of the first finds the row by itself (a gather of two
// floats a draft).

// Four neighbouring weights of the row, from v on; classes past its end weigh nothing.
struct Four {
  double w[4];
};
__device__ __forceinline__ Four weights(const Row& r, int64_t v, int64_t vocab, bool left) {
  f4 p = {0.f, 0.f, 0.f, 0.f}, q = p;
  if (v + 4 <= vocab) {
    p = *reinterpret_cast<const f4u*>(r.p + v);
    if (left && r.q) q = *reinterpret_cast<const f4u*>(r.q + v);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (v + j < vocab) {
        p[j] = r.p[v + j];
        if (left && r.q) q[j] = r.q[v + j];
      }
  }
  Four f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const double d = (double)p[j] - (double)q[j];
    f.w[j] = d > 0.0 && !(left && v + j == r.removed) ? d : 0.0;
  }
  return f;
}

// A chunk's weights: what the draft leaves, and the target's own.
struct Sums {
  double left, own;
};

template <int U>
__global__ __launch_bounds__(NT) void verify_sums_k(const VerifyArgs g, Sums* __restrict__ part) {
  __shared__ unsigned long long slot;
  __shared__ double red[NT / 64];
  const int64_t b = blockIdx.y;
  bool rejected;
  const int64_t kept = count_kept<NT>(g, b, &slot, rejected);
  if (blockIdx.x == 0 && threadIdx.x == 0) g.accepted[b] = kept;
  const Row r = row_of(g, b, kept, rejected);
  const int64_t v0 = (int64_t)blockIdx.x * (NT * 4 * U);
  double own = 0.0, left = 0.0;
  f4 p[U], q[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t v = v0 + (int64_t)(u * NT + threadIdx.x) * 4;
    p[u] = q[u] = f4{0.f, 0.f, 0.f, 0.f};
    if (v + 4 <= g.vocab) {
      p[u] = *reinterpret_cast<const f4u*>(r.p + v);
      if (r.q) q[u] = *reinterpret_cast<const f4u*>(r.q + v);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v + j < g.vocab) {
          p[u][j] = r.p[v + j];
          if (r.q) q[u][j] = r.q[v + j];
        }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t v = v0 + (int64_t)(u * NT + threadIdx.x) * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double pd = p[u][j] > 0.f ? (double)p[u][j] : 0.0;
      const double d = (double)p[u][j] - (double)q[u][j];
      own += pd;
      left += d > 0.0 && v + j != r.removed ? d : 0.0;
    }
  }
  own = block_sum<NT>(own, red);
  left = block_sum<NT>(left, red);
  if (threadIdx.x == 0) part[b * gridDim.x + blockIdx.x] = Sums{left, own};
}

// chunk: classes a chunk; chunks: of them.
__global__ __launch_bounds__(NT) void verify_pick_k(const VerifyArgs g, const Sums* __restrict__ part, int64_t chunk,
                                                    int64_t chunks) {
  __shared__ double red[NT / 64];
  __shared__ unsigned long long found;
  __shared__ long long last;
  __shared__ double base;
  const int64_t b = blockIdx.x;
  const int t = threadIdx.x;
  const int64_t kept = g.accepted[b];
  int64_t len = g.lengths ? g.lengths[b] : g.drafts;
  len = min(max(len, (int64_t)0), g.drafts);
  const bool rejected = kept < len;
  const Row r = row_of(g, b, kept, rejected);
  const Sums* pb = part + b * chunks;
  double own = 0.0, left = 0.0;
  for (int64_t i = t; i < chunks; i += NT) {
    left += pb[i].left;
    own += pb[i].own;
  }
  own = block_sum<NT>(own, red);
  left = block_sum<NT>(left, red);
  const bool use_left = rejected && left > 0.0;
  const double limit = (double)g.uniforms[b * (g.drafts + 1) + g.drafts] * (use_left ? left : own);
  if (t == 0) {
    found = ~0ull;
    last = -1;
    base = 0.0;
  }
  __syncthreads();
  // the first chunk whose end is past the limit, or the last one with weight
  double carry = 0.0;
  for (int64_t i0 = 0; i0 < chunks; i0 += NT) {
    const int64_t i = i0 + t;
    const double w = i < chunks ? (use_left ? pb[i].left : pb[i].own) : 0.0;
    double all;
    const double before = carry + block_before<NT>(w, red, all);
    if (w > 0.0) {
      if (before + w > limit) atomicMin(&found, (unsigned long long)i);
      atomicMax(&last, (long long)i);
    }
    __syncthreads();
    const unsigned long long f = found;
    if (f != ~0ull ? f == (unsigned long long)i : i == last) base = before;
    __syncthreads();
    if (f != ~0ull) break;
    carry += all;
  }
  const int64_t at = found != ~0ull ? (int64_t)found : last;
  int64_t token = -1;
  if (at >= 0) {
    carry = base;
    __syncthreads();
    if (t == 0) {
      found = ~0ull;
      last = -1;
    }
    __syncthreads();
    const int64_t end = min((at + 1) * chunk, g.vocab);
    for (int64_t v0 = at * chunk; v0 < end; v0 += NT * 4) {
      const int64_t v = v0 + t * 4;
      const Four f = weights(r, v, g.vocab, use_left);
      double all;
      double run = carry + block_before<NT>((f.w[0] + f.w[1]) + (f.w[2] + f.w[3]), red, all);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (f.w[j] > 0.0) {
          run += f.w[j];
          if (run > limit) atomicMin(&found, (unsigned long long)(v + j));
          atomicMax(&last, (long long)(v + j));
        }
      carry += all;
      __syncthreads();
      if (found != ~0ull) break;
    }
    token = found != ~0ull ? (int64_t)found : (int64_t)last;
  }
  for (int64_t i = t; i <= g.drafts; i += NT)
    g.out[b * (g.drafts + 1) + i] = i < kept ? g.tokens[b * g.drafts + i] : i == kept ? token : -1;
}

// Float4s a thread of the first launch: as many as leave two blocks a CU, so that
// a small batch's rows are cut finer.
int64_t chunk_units(int64_t batch, int64_t vocab) {
  int64_t u = 8;
  while (u > 1 && batch * ceil_div(vocab, NT * 4 * u) < 512) u /= 2;
  return u;
}

}  // namespace
}  // namespace oxi

using namespace oxi;

extern "C" {

int oxi_verify_drafts_workspace(int64_t batch, int64_t vocab, int64_t* bytes) {
  if (batch < 0 || vocab < 0) return fail(OXI_INVALID_ARGUMENT, "verify_drafts_workspace: negative size");
  if (vocab > ((int64_t)1 << 30) || batch > 65535)
    return fail(OXI_INVALID_ARGUMENT, "verify_drafts_workspace: size exceeds the kernel limits");
  if (!bytes) return fail(OXI_INVALID_ARGUMENT, "verify_drafts_workspace: NULL result pointer");
  *bytes = vocab > 0 ? batch * ceil_div(vocab, NT * 4 * chunk_units(batch, vocab)) * (int64_t)sizeof(Sums) : 0;
  return OXI_OK;
}

int oxi_verify_drafts(const float* target, const float* draft, const int64_t* tokens, const int64_t* lengths,
                      const float* uniforms, int64_t* accepted, int64_t* out, void* workspace, int64_t batch,
                      int64_t drafts, int64_t vocab) {
  if (batch < 0 || drafts < 0 || vocab < 0) return fail(OXI_INVALID_ARGUMENT, "verify_drafts: negative size");
  if (vocab > ((int64_t)1 << 30) || batch > 65535 || drafts > ((int64_t)1 << 20))
    return fail(OXI_INVALID_ARGUMENT, "verify_drafts: size exceeds the kernel limits");
  if (batch == 0) return OXI_OK;
  if (vocab == 0) return fail(OXI_INVALID_ARGUMENT, "verify_drafts: zero classes");
  if (!target || (drafts && !tokens) || !uniforms || !accepted || !out)
    return fail(OXI_INVALID_ARGUMENT, "verify_drafts: NULL tensor pointer");
  if (reinterpret_cast<uintptr_t>(workspace) & 7u)
    return fail(OXI_INVALID_ARGUMENT, "verify_drafts: the workspace at %p is not 8-byte aligned", workspace);
  OXI_CHECK_INIT();
  const VerifyArgs g{target, draft, tokens, lengths, uniforms, accepted, out, batch, drafts, vocab, guard_flag()};
  const int64_t u = chunk_units(batch, vocab), chunk = NT * 4 * u, chunks = ceil_div(vocab, chunk);
  Workspace ws(workspace ? 0 : sizeof(Sums) * (size_t)(batch * chunks));
  Sums* part = workspace ? static_cast<Sums*>(workspace) : ws.as<Sums>();
  if (!part) return fail_alloc("verify_drafts: sums");
  const dim3 grid((unsigned)chunks, (unsigned)batch);
  switch (u) {
    case 1: verify_sums_k<1><<<grid, dim3(NT), 0, stream()>>>(g, part); break;
    case 2: verify_sums_k<2><<<grid, dim3(NT), 0, stream()>>>(g, part); break;
    case 4: verify_sums_k<4><<<grid, dim3(NT), 0, stream()>>>(g, part); break;
    default: verify_sums_k<8><<<grid, dim3(NT), 0, stream()>>>(g, part);
  }
  if (int rc = check_launch("verify_drafts")) return rc;
  verify_pick_k<<<dim3((unsigned)batch), dim3(NT), 0, stream()>>>(g, part, chunk, chunks);
  return check_launch("verify_drafts");
}

}  // extern "C"

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

// A draft's probability: what a negative one stands for is 0 (a NaN stays).
__device__ __forceinline__ float drafted(float q) { return q < 0.f ? 0.f : q; }

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
      const double q = g.draft ? (double)drafted(g.draft[(b * g.drafts + i) * g.vocab + x]) : 1.0;
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

// A piece's weights: what the draft leaves, and the target's own.
struct Sums {
  double left, own;
};

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

// The same of two sums at once.
template <int N>
__device__ __forceinline__ Sums block_before(Sums v, Sums* lds, Sums& all) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  Sums s = v;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const double l = __shfl_up(s.left, m, 64), o = __shfl_up(s.own, m, 64);
    if (lane >= m) {
      s.left += l;
      s.own += o;
    }
  }
  __syncthreads();
  if (lane == 63) lds[wid] = s;
  __syncthreads();
  Sums base = {0.0, 0.0};
  all = {0.0, 0.0};
#pragma unroll
  for (int i = 0; i < N / 64; ++i) {
    if (i < wid) {
      base.left += lds[i].left;
      base.own += lds[i].own;
    }
    all.left += lds[i].left;
    all.own += lds[i].own;
  }
  return {base.left + (s.left - v.left), base.own + (s.own - v.own)};
}

// ---------------------------------------------------------------------------
// Two launches: the first cuts each sequence's row into pieces of 64 lanes x U
// float4s, a wave a piece, which sums its weights; the second, a block a
// sequence, finds the piece that the drawn number falls into and reads that
// one again. Each block of the first finds the row by itself (a gather of two
// floats a draft). HBM bounds the first, behind the three dependent loads that find the
// row: 128 sequences of 131072 classes, of which half reject a token, 100 MB in 20.3
// us, 4.9 TB/s (a block a sequence walking its row: 810); the second takes 5.9 us
// there, a chain of dependent loads and scans. 4 sequences of 32000: 3.7 and 3.9 us,
// both such chains.

template <int U>
__global__ __launch_bounds__(NT) void verify_sums_k(const VerifyArgs g, Sums* __restrict__ part, int64_t pieces) {
  __shared__ unsigned long long slot;
  const int64_t b = blockIdx.y;
  bool rejected;
  const int64_t kept = count_kept<NT>(g, b, &slot, rejected);
  if (blockIdx.x == 0 && threadIdx.x == 0) g.accepted[b] = kept;
  const Row r = row_of(g, b, kept, rejected);
  const int64_t piece = (int64_t)blockIdx.x * (NT / 64) + (threadIdx.x >> 6);
  const int64_t v0 = piece * (256 * U) + (threadIdx.x & 63) * 4;
  double own = 0.0, left = 0.0;
  f4 p[U], q[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t v = v0 + u * 256;
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
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double pd = p[u][j] > 0.f ? (double)p[u][j] : 0.0;
      const double d = (double)p[u][j] - (double)drafted(q[u][j]);
      own += pd;
      left += d > 0.0 && v0 + u * 256 + j != r.removed ? d : 0.0;
    }
  }
  own = wave_sum<double>(own);
  left = wave_sum<double>(left);
  if ((threadIdx.x & 63) == 0 && piece < pieces) part[b * pieces + piece] = Sums{left, own};
}

// The first thread with weight at whose weight the running sum, a thread's weight
// after those before it, passes `limit`, and the sum before it; -1 where it passes
// none's. The first, and not the one whose own stretch holds the limit: sums that
// end one stretch and begin the next are rounded apart, so that a limit there lies
// in both or in neither.
struct Crossing {
  int at;
  double before;
};
template <int N>
__device__ __forceinline__ Crossing cross(double w, double before, double limit, Crossing* slots) {
  const bool over = w > 0.0 && before + w > limit;
  const uint64_t lanes = __ballot(over);
  const int lane = threadIdx.x & 63, first = lanes ? __builtin_ctzll(lanes) : 0;
  __syncthreads();
  if (lane == first) slots[threadIdx.x >> 6] = {over ? (int)threadIdx.x : -1, before};
  __syncthreads();
  Crossing c = {-1, 0.0};
#pragma unroll
  for (int i = N / 64 - 1; i >= 0; --i)
    if (slots[i].at >= 0) c = slots[i];
  return c;
}

// U: as in the first launch, the classes of a piece that each thread has.
template <int U>
__global__ __launch_bounds__(NT) void verify_pick_k(const VerifyArgs g, const Sums* __restrict__ part, int64_t pieces) {
  static_assert(NT == 256, "a piece is 256 U classes");
  __shared__ double red[NT / 64];
  __shared__ Sums both[NT / 64];
  __shared__ Crossing slots[NT / 64];
  __shared__ int last;
  const int64_t b = blockIdx.x;
  const int t = threadIdx.x;
  const int64_t kept = g.accepted[b];
  int64_t len = g.lengths ? g.lengths[b] : g.drafts;
  len = min(max(len, (int64_t)0), g.drafts);
  const bool rejected = kept < len;
  const Row r = row_of(g, b, kept, rejected);
  const double u = (double)g.uniforms[b * (g.drafts + 1) + g.drafts];
  const Sums* pb = part + b * pieces;
  // both kinds' sums over the first NT pieces, which are all of most vocabularies
  const Sums mine0 = t < pieces ? pb[t] : Sums{0.0, 0.0};
  Sums total;
  const Sums before0 = block_before<NT>(mine0, both, total);
  const Sums first = total;
  if (pieces > NT) {
    double left = 0.0, own = 0.0;
    for (int64_t i = NT + t; i < pieces; i += NT) {
      left += pb[i].left;
      own += pb[i].own;
    }
    total.left += block_sum<NT>(left, red);
    total.own += block_sum<NT>(own, red);
  }
  const bool use_left = rejected && total.left > 0.0;
  // a number that is not below 1 draws the last class, whatever the sums' roundings
  double limit = u < 1.0 ? u * (use_left ? total.left : total.own) : (double)__builtin_huge_valf();
  // the piece
  const Crossing c0 = cross<NT>(use_left ? mine0.left : mine0.own, use_left ? before0.left : before0.own, limit, slots);
  int64_t at = c0.at;
  double base = c0.before, carry = use_left ? first.left : first.own;
  for (int64_t i0 = NT; at < 0 && i0 < pieces; i0 += NT) {
    const double w = i0 + t < pieces ? (use_left ? pb[i0 + t].left : pb[i0 + t].own) : 0.0;
    double all;
    const double before = carry + block_before<NT>(w, red, all);
    const Crossing c = cross<NT>(w, before, limit, slots);
    if (c.at >= 0) {
      at = i0 + c.at;
      base = c.before;
      break;
    }
    carry += all;
  }
  if (at < 0 && carry > 0.0) {  // the last piece with weight
    for (int64_t i0 = (pieces - 1) / NT * NT; i0 >= 0 && at < 0; i0 -= NT) {
      __syncthreads();
      if (t == 0) last = -1;
      __syncthreads();
      if (i0 + t < pieces && (use_left ? pb[i0 + t].left : pb[i0 + t].own) > 0.0) atomicMax(&last, t);
      __syncthreads();
      if (last >= 0) at = i0 + last;
    }
    limit = (double)__builtin_huge_valf();  // in it the last class with weight, not the first past the limit
  }
  int64_t token = -1;
  if (at >= 0) {
    // a thread's U neighbouring classes
    const int64_t v0 = at * (256 * U) + (int64_t)t * U;
    float p[U], q[U];
    if (v0 + U <= g.vocab) {
      typedef float V __attribute__((ext_vector_type(U < 4 ? U : 4), aligned(4)));
      constexpr int W = U < 4 ? U : 4;
#pragma unroll
      for (int k = 0; k < U; k += W) {
        const V pv = *reinterpret_cast<const V*>(r.p + v0 + k);
        V qv = {};
        if (use_left && r.q) qv = *reinterpret_cast<const V*>(r.q + v0 + k);
#pragma unroll
        for (int j = 0; j < W; ++j) {
          p[k + j] = pv[j];
          q[k + j] = qv[j];
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < U; ++j) {
        p[j] = v0 + j < g.vocab ? r.p[v0 + j] : 0.f;
        q[j] = v0 + j < g.vocab && use_left && r.q ? r.q[v0 + j] : 0.f;
      }
    }
    auto weight = [&](int j) {
      const double d = (double)p[j] - (double)drafted(q[j]);
      return d > 0.0 && !(use_left && v0 + j == r.removed) ? d : 0.0;
    };
    double w = 0.0;
    int mine = -1;  // this thread's last class with weight
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const double x = weight(j);
      w += x;
      if (x > 0.0) mine = j;
    }
    double all;
    const double before = base + block_before<NT>(w, red, all);
    Crossing c = cross<NT>(w, before, limit, slots);
    if (c.at < 0) {  // the last thread with weight, its last class
      if (t == 0) last = -1;
      __syncthreads();
      if (mine >= 0) atomicMax(&last, t);
      __syncthreads();
      c.at = last;
    }
    if (t == c.at) {
      double run = before;
      int hit = -1;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const double x = weight(j);
        run += x;
        if (hit < 0 && x > 0.0 && run > limit) hit = j;
      }
      token = v0 + (hit >= 0 ? hit : mine);
    } else {
      token = -2;  // another thread's
    }
  }
  if (token != -2 && (at >= 0 || t == 0)) g.out[b * (g.drafts + 1) + kept] = token;
  for (int64_t i = t; i <= g.drafts; i += NT)
    if (i != kept) g.out[b * (g.drafts + 1) + i] = i < kept ? g.tokens[b * g.drafts + i] : -1;
}

int64_t pieces_of(int64_t vocab, int64_t u) { return ceil_div(vocab, 256 * u); }

// Float4s a thread of the first launch: as many as leave two blocks a CU, so that
// a small batch's rows are cut finer.
int64_t piece_units(int64_t batch, int64_t vocab) {
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
  *bytes = vocab > 0 ? batch * pieces_of(vocab, piece_units(batch, vocab)) * (int64_t)sizeof(Sums) : 0;
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
  const int64_t u = piece_units(batch, vocab), pieces = pieces_of(vocab, u);
  Workspace ws(workspace ? 0 : sizeof(Sums) * (size_t)(batch * pieces));
  Sums* part = workspace ? static_cast<Sums*>(workspace) : ws.as<Sums>();
  if (!part) return fail_alloc("verify_drafts: sums");
  const dim3 grid((unsigned)ceil_div(pieces, NT / 64), (unsigned)batch);
#define OXI_VER(U)                                                                            \
  verify_sums_k<U><<<grid, dim3(NT), 0, stream()>>>(g, part, pieces);                                \
  if (int rc = check_launch("verify_drafts")) return rc;                                     \
  verify_pick_k<U><<<dim3((unsigned)batch), dim3(NT), 0, stream()>>>(g, part, pieces);
  switch (u) {
    case 1: OXI_VER(1) break;
    case 2: OXI_VER(2) break;
    case 4: OXI_VER(4) break;
    default: OXI_VER(8)
  }
#undef OXI_VER
  return check_launch("verify_drafts");
}

}  // extern "C"

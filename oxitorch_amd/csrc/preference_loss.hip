// The preference loss of pairs of sequences (chosen, rejected) over rows of logits,
// and its gradient. With S the sum (or the mean) of logp over a sequence's counted
// tokens, R the same of the reference's,
//
//   u = beta ((S_c - R_c) - (S_r - R_r)) - margin
//   sigmoid: (1 - e) softplus(-u) + e softplus(u);  hinge: max(0, 1 - u);
//   ipo: (u/beta - 1/(2 beta))^2
//   loss = sum over the pairs / pairs
//   d loss/d logp = +- beta f'(u)/pairs (/ count for the mean) for each token
//
// (logp and its gradient: token_rows.h). A gradient needs its whole pair's sums, so the
// logits are read twice. Log-probabilities are summed in 64 bits: a difference of
// sums over hundreds of tokens decides.
#include <cmath>

#include "token_rows.h"

namespace oxi {
namespace {

struct PreferenceOp {
  static constexpr int READ_MAX = ROWS_MAX_READ;
  double* logp;
  float *coef, *saved;
  struct Given {};
  __device__ __forceinline__ Given load(int64_t) const { return {}; }
  __device__ __forceinline__ Two finish(int64_t row, const Given&, const RowStats& r, bool lead) const {
    if (!lead) return {0.f, 0.f};
    logp[row] = r.logp;
    coef[row] = 0.f;  // a counted row's own comes with its pair
    save_row(saved, row, r);
    return {0.f, 0.f};
  }
  __device__ __forceinline__ void skip(int64_t row) const {
    logp[row] = 0.0;
    coef[row] = 0.f;
    save_nothing(saved, row);
  }
};

struct PairArgs {
  const int64_t* starts;
  const int64_t* ids;
  const double* logp;
  const float* ref;
  float *pair_loss, *seq_logp, *coef;
  int64_t n, pairs;
  int c, kind, average;
  double beta, margin, smoothing;
  int* guard;
};

// log(1 + e^x)
__device__ __forceinline__ double softplus(double x) { return (x > 0.0 ? x : 0.0) + log1p64(exp64(-fabs(x))); }

constexpr int PAIR_NT = 256;

// A block a pair.
__global__ __launch_bounds__(PAIR_NT) void preference_pair_k(const PairArgs g) {
  __shared__ double red[PAIR_NT / 64];
  const int64_t p = blockIdx.x;
  double sum[2], own[2], count[2];
  int64_t first[2], last[2];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    int64_t a = g.starts[2 * p + side], b = g.starts[2 * p + side + 1];
    if (a < 0 || b < a || b > g.n) {  // such a sequence is empty
      if (threadIdx.x == 0) atomicOr(g.guard, 1);
      a = b = 0;
    }
    first[side] = a;
    last[side] = b;
    double s = 0.0, r = 0.0, k = 0.0;
    for (int64_t i = a + threadIdx.x; i < b; i += PAIR_NT) {
      const int64_t id = g.ids[i];
      if (id < 0 || id >= g.c) continue;
      s += g.logp[i];
      if (g.ref) r += (double)g.ref[i];
      k += 1.0;
    }
    s = block_sum<PAIR_NT>(s, red);
    r = block_sum<PAIR_NT>(r, red);
    k = block_sum<PAIR_NT>(k, red);
    count[side] = g.average ? fmax(k, 1.0) : 1.0;
    own[side] = s / count[side];
    sum[side] = (s - r) / count[side];
  }
  const double u = g.beta * (sum[0] - sum[1]) - g.margin;
  double loss, slope;  // slope: of loss by the log-ratio
  if (g.kind == OXI_PREFERENCE_SIGMOID) {
    const double e = exp64(-fabs(u));
    const double above = (u > 0.0 ? 1.0 : e) / (1.0 + e);  // sigmoid(u)
    const double below = (u > 0.0 ? e : 1.0) / (1.0 + e);
    loss = (1.0 - g.smoothing) * softplus(-u) + (g.smoothing != 0.0 ? g.smoothing * softplus(u) : 0.0);
    slope = g.beta * (g.smoothing * above - (1.0 - g.smoothing) * below);
  } else if (g.kind == OXI_PREFERENCE_HINGE) {
    loss = u < 1.0 ? 1.0 - u : u != u ? u : 0.0;
    slope = u < 1.0 ? -g.beta : u != u ? u : 0.0;
  } else {
    const double d = (u - 0.5) / g.beta;
    loss = d * d;
    slope = 2.0 * d;
  }
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const float k = (float)((side ? -slope : slope) / ((double)g.pairs * count[side]));
    for (int64_t i = first[side] + threadIdx.x; i < last[side]; i += PAIR_NT) {
      const int64_t id = g.ids[i];
      if (id >= 0 && id < g.c) g.coef[i] = k;
    }
  }
  if (threadIdx.x == 0) {
    g.pair_loss[p] = (float)loss;
    g.seq_logp[2 * p] = (float)own[0];
    g.seq_logp[2 * p + 1] = (float)own[1];
  }
}

__global__ __launch_bounds__(PAIR_NT) void preference_mean_k(const float* __restrict__ pair_loss, int64_t pairs,
                                                             float* __restrict__ loss) {
  __shared__ double red[PAIR_NT / 64];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < pairs; i += PAIR_NT) s += (double)pair_loss[i];
  s = block_sum<PAIR_NT>(s, red);
  if (threadIdx.x == 0) loss[0] = (float)(s / (double)pairs);
}

int64_t workspace_bytes(int64_t n, int64_t c) { return token_parts_bytes(n, c) + n * (int64_t)sizeof(double); }

int check_preference(const char* what, int64_t n, int64_t c, int64_t pairs) {
  if (int rc = check_token_rows(what, n, c, 1.f)) return rc;
  if (pairs < 0) return fail(OXI_INVALID_ARGUMENT, "%s: negative size", what);
  if (!grid_fits(pairs, 1024)) return fail(OXI_INVALID_ARGUMENT, "%s: size exceeds the kernel limits", what);
  return OXI_OK;
}

}  // namespace
}  // namespace oxi

using namespace oxi;

extern "C" {

int oxi_preference_loss_workspace(int64_t n, int64_t c, int64_t* bytes) {
  if (!bytes) return fail(OXI_INVALID_ARGUMENT, "preference_loss_workspace: NULL result");
  if (int rc = check_token_rows("preference_loss_workspace", n, c, 1.f)) return rc;
  *bytes = workspace_bytes(n, c);
  return OXI_OK;
}

int oxi_preference_loss_fwd(const float* logits, const int64_t* ids, const int64_t* starts, const float* ref_logp,
                            float* loss, float* pair_loss, float* seq_logp, float* coef, float* saved, float* dlogits,
                            void* workspace, int64_t n, int64_t c, int64_t pairs, int kind, int average, float beta,
                            float margin, float smoothing) {
  const char* what = "preference_loss_fwd";
  if (int rc = check_preference(what, n, c, pairs)) return rc;
  if (kind != OXI_PREFERENCE_SIGMOID && kind != OXI_PREFERENCE_HINGE && kind != OXI_PREFERENCE_IPO)
    return fail(OXI_INVALID_ARGUMENT, "%s: unknown kind %d", what, kind);
  if (!(beta > 0.f) || std::isinf(beta))
    return fail(OXI_INVALID_ARGUMENT, "%s: beta must be positive, got %g", what, (double)beta);
  if (!std::isfinite(margin)) return fail(OXI_INVALID_ARGUMENT, "%s: the margin must be finite", what);
  if (!(smoothing >= 0.f && smoothing < 1.f))
    return fail(OXI_INVALID_ARGUMENT, "%s: the smoothing must lie in [0, 1), got %g", what, (double)smoothing);
  if (smoothing != 0.f && kind != OXI_PREFERENCE_SIGMOID)
    return fail(OXI_INVALID_ARGUMENT, "%s: smoothing goes with the sigmoid kind", what);
  if (!loss) return fail(OXI_INVALID_ARGUMENT, "%s: loss must not be NULL", what);
  if (pairs && (!starts || !pair_loss || !seq_logp)) return fail(OXI_INVALID_ARGUMENT, "%s: NULL tensor pointer", what);
  if (n && (!logits || !ids || !coef || !saved || !starts))
    return fail(OXI_INVALID_ARGUMENT, "%s: NULL tensor pointer", what);
  if (reinterpret_cast<uintptr_t>(workspace) & 15)
    return fail(OXI_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", what);
  OXI_CHECK_INIT();
  Workspace own(workspace ? 0 : (size_t)workspace_bytes(n, c));
  if (n && !workspace && !own.p) return fail_alloc(what);
  f4* parts = static_cast<f4*>(workspace ? workspace : own.p);
  double* logp = reinterpret_cast<double*>(parts + token_parts_bytes(n, c) / (int64_t)sizeof(f4));
  if (n) {
    TokenRows in = token_rows(logits, ids, n, c, 1.f);
    in.starts = starts;
    in.sequences = 2 * pairs;
    in.again = true;
    if (int rc = token_rows_read(in, parts, PreferenceOp{logp, coef, saved}, what)) return rc;
  }
  if (pairs) {
    const PairArgs g{starts, ids, logp, ref_logp, pair_loss, seq_logp, coef, n, pairs, (int)c, kind, average ? 1 : 0,
                     (double)beta, (double)margin, (double)smoothing, guard_flag()};
    preference_pair_k<<<dim3((unsigned)pairs), dim3(PAIR_NT), 0, stream()>>>(g);
    if (int rc = check_launch(what)) return rc;
    preference_mean_k<<<1, PAIR_NT, 0, stream()>>>(pair_loss, pairs, loss);
    if (int rc = check_launch(what)) return rc;
  } else if (int rc = oxi_fill(loss, 1, 0.f)) {
    return rc;
  }
  if (n && dlogits) return launch_token_bwd(logits, ids, saved, coef, nullptr, nullptr, dlogits, n, c, 1.f, what);
  return OXI_OK;
}

}  // extern "C"

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
  static constexpr bool SUMMED = true;
  static constexpr bool SAME_BITS = false;  // there is one way
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
  TokenRows in;
  const f4* parts;     // the rows' parts, np each; NULL: their log-probabilities are in logp
  const double* logp;
  int np;
  const float* ref;
  float *pair_loss, *seq_logp, *coef, *saved;
  int64_t pairs;
  int kind, average;
  double beta, margin, smoothing;
};

// log(1 + e^x)
__device__ __forceinline__ double softplus(double x) { return (x > 0.0 ? x : 0.0) + log1p64(exp64(-fabs(x))); }

// Threads of a pair's block, half of them to each sequence; the most parts a row of rows that
// they join, a row a thread. That saves a launch: when rows of 32000 classes came by parts too, 92 of
// them in 2 pairs took 7 us here, and 10.5 with a wave a row in a launch of its own, 256 threads a
// pair and a launch for the mean.
constexpr int PAIR_NT = 1024, HALF = PAIR_NT / 2, JOIN_MOST = 16;

// A block a pair.
__global__ __launch_bounds__(PAIR_NT) void preference_pair_k(const PairArgs g) {
  __shared__ double red[3 * (PAIR_NT / 64)];
  const TokenRows& in = g.in;
  const int t = threadIdx.x;
  const int64_t p = blockIdx.x;
  const int side = t / HALF;
  int64_t first = in.starts[2 * p + side], last = in.starts[2 * p + side + 1];
  if (first < 0 || last < first || last > in.n) {  // such a sequence is empty
    if ((t & (HALF - 1)) == 0) atomicOr(in.guard, 1);
    first = last = 0;
  }
  double s = 0.0, r = 0.0, k = 0.0;
  for (int64_t i = first + (t & (HALF - 1)); i < last; i += HALF) {
    const int64_t id = in.ids[i];
    if (!in.counts(i, id)) continue;
    if (g.ref) r += (double)g.ref[i];
    if (g.parts) {
      const RowStats row = joined_row(in, g.parts + i * g.np, g.np, in.x[i * in.c + id]);
      save_row(g.saved, i, row);
      s += row.logp;
    } else {
      s += g.logp[i];
    }
    k += 1.0;
  }
  s = over_block<64, AddF64>(s, (double*)nullptr);
  r = over_block<64, AddF64>(r, (double*)nullptr);
  k = over_block<64, AddF64>(k, (double*)nullptr);
  if ((t & 63) == 0) {
    red[3 * (t >> 6)] = s;
    red[3 * (t >> 6) + 1] = r;
    red[3 * (t >> 6) + 2] = k;
  }
  __syncthreads();
  double sum[2], own[2], count[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    double v[3] = {0.0, 0.0, 0.0};
#pragma unroll
    for (int w = 0; w < HALF / 64; ++w)
#pragma unroll
      for (int i = 0; i < 3; ++i) v[i] += red[3 * (q * (HALF / 64) + w) + i];
    count[q] = g.average ? fmax(v[2], 1.0) : 1.0;
    own[q] = v[0] / count[q];
    sum[q] = (v[0] - v[1]) / count[q];
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
  const float by = (float)((side ? -slope : slope) / ((double)g.pairs * (side ? count[1] : count[0])));
  for (int64_t i = first + (t & (HALF - 1)); i < last; i += HALF)
    if (in.counts(i, in.ids[i])) g.coef[i] = by;
  if (t == 0) {
    g.pair_loss[p] = (float)loss;
    g.seq_logp[2 * p] = (float)own[0];
    g.seq_logp[2 * p + 1] = (float)own[1];
  }
}

__global__ __launch_bounds__(MEAN_NT) void preference_mean_k(const MeanOf mean) { mean.by_block(); }

// The parts' sums and the log-probabilities.
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
  if (n && dlogits == logits) return fail(OXI_INVALID_ARGUMENT, "%s: dlogits must not be the logits", what);
  OXI_CHECK_INIT();
  Workspace own(workspace ? 0 : (size_t)workspace_bytes(n, c));
  if (n && !workspace && !own.p) return fail_alloc(what);
  if (!pairs) {
    if (int rc = oxi_fill(loss, 1, 0.f)) return rc;
  }
  f4* parts = static_cast<f4*>(workspace ? workspace : own.p);
  double* logp = reinterpret_cast<double*>(parts + token_parts_bytes(n, c) / (int64_t)sizeof(f4));
  TokenRows in = token_rows(logits, ids, n, c, 1.f);
  in.starts = starts;
  in.sequences = 2 * pairs;
  in.coef = coef;
  in.saved = saved;
  const int np = (int)row_parts(c);
  const bool by_pairs = c > ROWS_MAX && np <= JOIN_MOST;
  if (n) {
    const int rc = by_pairs ? launch_token_parts(in, parts, what)
                            : token_rows_read(in, parts, PreferenceOp{logp, coef, saved}, what);
    if (rc) return rc;
  }
  if (pairs) {
    const PairArgs g{in, by_pairs ? parts : nullptr, logp, np, ref_logp, pair_loss, seq_logp, coef, saved, pairs, kind, average ? 1 : 0, (double)beta, (double)margin, (double)smoothing};
    preference_pair_k<<<dim3((unsigned)pairs), dim3(PAIR_NT), 0, stream()>>>(g);
    if (int rc = check_launch(what)) return rc;
  }
  const MeanOf mean{pair_loss, pairs, loss};
  if (n && dlogits)  // one of its blocks takes the mean
    return launch_token_bwd(logits, ids, saved, coef, nullptr, nullptr, dlogits, n, c, 1.f, what, mean);
  if (!pairs) return OXI_OK;
  preference_mean_k<<<1, MEAN_NT, 0, stream()>>>(mean);
  return check_launch(what);
}

}  // extern "C"

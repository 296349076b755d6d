// The clipped policy loss over rows of logits with a KL term and an entropy bonus,
// and its gradient. For a row's chosen token, with r = exp(logp - old) and the
// advantage A:
//
//   s = min(r A, clip(r, 1 - low, 1 + high) A), for A < 0 at least most A
//   k = e^d - 1 - d, d = ref - logp
//   row = -s + kl k - ent H,   loss = sum w row / divisor
//   d row/d logp = -[s is r A] r A - kl (e^d - 1),   d row/d H = -ent
//
// (the mathematics of logp, H and their gradients is in token_rows.h). All of a row's
// own arithmetic is in 64 bits: k of a policy near its reference is the small rest of
// terms that cancel, and a ratio next to an edge of the clipping must fall on the side
// that the definition has it on.
#include <cmath>

#include "token_rows.h"

namespace oxi {
namespace {

struct PolicyOp {
  static constexpr bool SUMMED = false;
  static constexpr bool SAME_BITS = true;  // with a gradient and without
  const float *adv, *old, *ref, *weights;
  float *rows, *logp, *coef, *saved;
  int64_t n;
  double low, high, most;  // the ratio's bounds, and the factor of a negative advantage that bounds s (0: none)
  double kl, ent, inv_div;

  // The row's own numbers, loaded before its logits.
  struct Given {
    float adv, old, ref, weight;
  };
  __device__ __forceinline__ Given load(int64_t row) const {
    return {adv[row], old ? old[row] : 0.f, ref ? ref[row] : 0.f, weights ? weights[row] : 1.f};
  }
  // Writes the row's results; the loss's derivatives by its logp and entropy.
  __device__ __forceinline__ Two finish(int64_t row, const Given& in, const RowStats& r, bool lead) const {
    const double A = (double)in.adv;
    const bool broken = r.logp != r.logp;  // the row holds no distribution: NaN whatever the ratio and the advantage
    const double ratio = broken ? r.logp : old ? exp64(r.logp - (double)in.old) : 1.0;
    const double free = A == 0.0 && !broken ? 0.0 : ratio * A;
    const double bounded = (ratio < low ? low : ratio > high ? high : ratio) * A;
    bool clipped = free > bounded;
    double s = clipped ? bounded : free;
    if (most > 0.0 && A < 0.0 && s < most * A) {
      s = most * A;
      clipped = true;
    }
    double g = clipped ? 0.0 : -free, k = 0.0;
    double loss = -s;
    if (ref) {
      const double d = (double)in.ref - r.logp;
      k = d == (double)__builtin_huge_valf() ? d : exp_rest(d);
      if (kl != 0.0) {
        g -= kl * (fabs(d) < 0.5 ? k + d : exp64(d) - 1.0);
        loss += kl * k;
      }
    }
    if (ent != 0.0) loss -= ent * r.entropy;
    const double w = (double)in.weight * inv_div;
    const Two by{(float)(g * w), (float)(-ent * w)};
    if (!lead) return by;
    rows[row] = (float)loss;
    rows[n + row] = (float)k;
    rows[2 * n + row] = (float)r.entropy;
    rows[3 * n + row] = clipped ? 1.f : 0.f;
    if (logp) logp[row] = (float)r.logp;
    coef[row] = by.a;
    coef[n + row] = by.b;
    save_row(saved, row, r);
    return by;
  }
  __device__ __forceinline__ void skip(int64_t row) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) rows[i * n + row] = 0.f;
    if (logp) logp[row] = 0.f;
    coef[row] = coef[n + row] = 0.f;
    save_nothing(saved, row);
  }
};

template <bool GRAD, bool ENT, bool NTS>
bool launch_as(const TokenRows& in, const PolicyOp& op, float* dx, void* workspace) {
  return launch_token_cluster<GRAD, ENT, NTS>(in, op, dx, workspace) || launch_token_rows_as<GRAD, ENT, NTS>(in, op, dx);
}

// One pass over the logits, the same with a gradient and without; false where no kernel holds such rows.
bool launch_rows(const TokenRows& in, const PolicyOp& op, float* dx, bool ent, void* workspace) {
  if (!dx) return launch_as<false, false, false>(in, op, dx, workspace);
  const bool nt = nt_stream_stores(in.n * in.c * 4);
  if (ent) return nt ? launch_as<true, true, true>(in, op, dx, workspace) : launch_as<true, true, false>(in, op, dx, workspace);
  return nt ? launch_as<true, false, true>(in, op, dx, workspace) : launch_as<true, false, false>(in, op, dx, workspace);
}

// The parts' sums, or a cluster's words, which are no more than the parts.
int64_t workspace_bytes(int64_t n, int64_t c) { return 64 + n * row_parts(c) * 3 * (int64_t)sizeof(uint64_t); }

// Four sums over a block of N threads, thread k < 4 returning the k-th: one barrier.
template <int N>
__device__ __forceinline__ double block_sums(const double (&acc)[4], double* red) {
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const double v = over_block<64, AddF64>(acc[k], (double*)nullptr);
    if ((threadIdx.x & 63) == 0) red[4 * wave + k] = v;
  }
  __syncthreads();
  double s = 0.0;
  if (threadIdx.x < 4)
#pragma unroll
    for (int w = 0; w < N / 64; ++w) s += red[4 * w + threadIdx.x];
  return s;
}

constexpr int MEAN_THREADS = 1024, MEAN_ROWS = 8192;  // rows a block

// The sums over each MEAN_ROWS rows, a block each in a fixed order: times `by` to out where there is one,
// else to parts. (8192 rows 5.5 us; the four sums one after another, a pair of barriers each, 6.5.)
__global__ __launch_bounds__(MEAN_THREADS) void policy_mean_k(const TokenRows in, const float* __restrict__ rows,
                                                              double by, float* __restrict__ out,
                                                              double* __restrict__ parts) {
  __shared__ double red[4 * (MEAN_THREADS / 64)];
  double acc[4] = {0.0, 0.0, 0.0, 0.0};
  constexpr int U = 4;  // rows in flight a thread
  const int64_t end = min(in.n, ((int64_t)blockIdx.x + 1) * MEAN_ROWS);
  for (int64_t i0 = (int64_t)blockIdx.x * MEAN_ROWS + threadIdx.x; i0 < end; i0 += U * MEAN_THREADS) {
    int64_t id[U];
    float w[U], v[4][U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = min(i0 + u * MEAN_THREADS, end - 1);
      id[u] = in.ids[i];
      w[u] = in.weights ? in.weights[i] : 1.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k][u] = rows[k * in.n + i];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u * MEAN_THREADS >= end || id[u] < 0 || id[u] >= in.c || w[u] == 0.f) continue;
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] += (double)w[u] * (double)v[k][u];
    }
  }
  const double s = block_sums<MEAN_THREADS>(acc, red);
  if (threadIdx.x >= 4) return;
  if (gridDim.x == 1) out[threadIdx.x] = (float)(s * by);
  else parts[4 * blockIdx.x + threadIdx.x] = s;
}

__global__ __launch_bounds__(256) void policy_mean_parts_k(const double* __restrict__ parts, int count, double by,
                                                           float* __restrict__ out) {
  __shared__ double red[4 * (256 / 64)];
  double acc[4] = {0.0, 0.0, 0.0, 0.0};
  for (int i = threadIdx.x; i < count; i += 256)
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] += parts[4 * i + k];
  const double s = block_sums<256>(acc, red);
  if (threadIdx.x < 4) out[threadIdx.x] = (float)(s * by);
}

}  // namespace
}  // namespace oxi

using namespace oxi;

extern "C" {

int oxi_policy_loss_workspace(int64_t n, int64_t c, int64_t* bytes) {
  if (!bytes) return fail(OXI_INVALID_ARGUMENT, "policy_loss_workspace: NULL result");
  if (int rc = check_token_rows("policy_loss_workspace", n, c, 1.f)) return rc;
  *bytes = n ? workspace_bytes(n, c) : 0;
  return OXI_OK;
}

int oxi_policy_loss_fwd(const float* logits, const int64_t* ids, const float* advantages, const float* old_logp,
                        const float* ref_logp, const float* weights, float* out, float* rows, float* logp, float* coef,
                        float* saved, float* dlogits, void* workspace, int64_t n, int64_t c, float temperature,
                        float clip_low, float clip_high, float clip_max, float kl_coef, float entropy_coef,
                        float divisor) {
  const char* what = "policy_loss_fwd";
  if (int rc = check_token_rows(what, n, c, temperature)) return rc;
  if (!(clip_low >= 0.f) || !(clip_high >= 0.f))
    return fail(OXI_INVALID_ARGUMENT, "%s: the clipping must not be negative, got %g and %g", what, (double)clip_low,
                (double)clip_high);
  if (clip_max != 0.f && !(clip_max >= 1.f))
    return fail(OXI_INVALID_ARGUMENT, "%s: clip_max must be 0 (none) or at least 1, got %g", what, (double)clip_max);
  if (!std::isfinite(kl_coef) || !std::isfinite(entropy_coef))
    return fail(OXI_INVALID_ARGUMENT, "%s: the coefficients must be finite", what);
  if (kl_coef != 0.f && !ref_logp)
    return fail(OXI_INVALID_ARGUMENT, "%s: a KL term needs the reference's log-probabilities", what);
  if (!(divisor > 0.f) || std::isinf(divisor))
    return fail(OXI_INVALID_ARGUMENT, "%s: the divisor must be positive, got %g", what, (double)divisor);
  if (!out) return fail(OXI_INVALID_ARGUMENT, "%s: out must not be NULL", what);
  if (n && (!logits || !ids || !advantages || !rows || !coef || !saved))
    return fail(OXI_INVALID_ARGUMENT, "%s: NULL tensor pointer", what);
  if (reinterpret_cast<uintptr_t>(workspace) & 15)
    return fail(OXI_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", what);
  if (n && dlogits == logits) return fail(OXI_INVALID_ARGUMENT, "%s: dlogits must not be the logits", what);
  OXI_CHECK_INIT();
  if (n == 0) return oxi_fill(out, 4, 0.f);
  Workspace own(workspace ? 0 : (size_t)workspace_bytes(n, c));
  if (!workspace && !own.p) return fail_alloc(what);
  TokenRows in = token_rows(logits, ids, n, c, temperature);
  in.weights = weights;
  const double inv_div = 1.0 / (double)divisor;
  const PolicyOp op{advantages, old_logp, ref_logp, weights, rows, logp, coef, saved, n, 1.0 - (double)clip_low,
                    1.0 + (double)clip_high, (double)clip_max, (double)kl_coef, (double)entropy_coef, inv_div};
  void* const at = workspace ? workspace : own.p;
  if (launch_rows(in, op, dlogits, entropy_coef != 0.f, at)) {
    if (int rc = check_launch(what)) return rc;
  } else {
    if (int rc = token_rows_by_parts(in, static_cast<f4*>(at), op, what)) return rc;
    if (dlogits)
      if (int rc = launch_token_bwd(logits, ids, saved, coef, entropy_coef != 0.f ? coef + n : nullptr, nullptr,
                                    dlogits, n, c, temperature, what))
        return rc;
  }
  // the rows' launches are done with the workspace, which holds more than the means' parts
  double* sums = static_cast<double*>(at);
  const int64_t blocks = ceil_div(n, MEAN_ROWS);
  policy_mean_k<<<dim3((unsigned)blocks), dim3(MEAN_THREADS), 0, stream()>>>(in, rows, inv_div, out, sums);
  if (blocks > 1) policy_mean_parts_k<<<1, 256, 0, stream()>>>(sums, (int)blocks, inv_div, out);
  return check_launch(what);
}

}  // extern "C"

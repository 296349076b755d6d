// Log-probabilities of chosen tokens and the entropies of the distributions they
// were chosen from, over rows of logits, with their gradient; the passes that the
// policy and preference losses share (the mathematics is in token_rows.h).
#include <cmath>
#include <cstdlib>
#include <cstring>

#include "token_rows.h"

namespace oxi {
namespace {

__global__ __launch_bounds__(PART_NT) void token_part_k(const TokenRows in, f4* __restrict__ parts, int np,
                                                        int64_t row0) {
  __shared__ float lds[3 * (PART_NT / 64)];
  const RowPiece of(blockIdx.x, gridDim.x / (unsigned)np, (unsigned)np);
  const int64_t row = row0 + of.row;
  const int part = of.piece;
  const int64_t id = in.ids[row];
  const int t = threadIdx.x;
  const bool counts = in.counts(row, id);
  if (part == 0 && t == 0) {
    if (in.coef) in.coef[row] = 0.f;
    if (in.saved && !counts) save_nothing(in.saved, row);
  }
  if (!counts) return;
  const float* xr = in.x + row * in.c;
  const RowLay<> lay(xr, in.c);
  const int at = lay.slot((int)id), comp = lay.component((int)id);
  const f4* x4 = reinterpret_cast<const f4*>(xr + lay.head);
  const int c0 = part * (PART_NT * PART_U) + t;
  f4 v[PART_U];
  float m = NEG_INF;
#pragma unroll
  for (int u = 0; u < PART_U; ++u) {
    const int q = c0 + u * PART_NT;
    v[u] = f4{NEG_INF, NEG_INF, NEG_INF, NEG_INF};
    if (q < lay.c4) v[u] = ld_stream(x4 + q);
  }
#pragma unroll
  for (int u = 0; u < PART_U; ++u)
    if (c0 + u * PART_NT == at) v[u] = drop(v[u], comp);
  const int e = part == 0 ? lay.edge(t, in.c) : -1;
  const float v1 = e >= 0 && e != (int)id ? xr[e] : NEG_INF;
#pragma unroll
  for (int u = 0; u < PART_U; ++u) m = fmaxf(m, max4(v[u]));
  m = over_block<PART_NT, MaxF32>(fmaxf(m, v1), lds);
  const float shift = m == NEG_INF ? 0.f : m;
  float s = 0.f, et = 0.f;
  auto add = [&](float x) {
    const float z = (x - shift) * in.scale2;
    const float p = __builtin_amdgcn_exp2f(z);
    s += p;
    et = fmaf(p, fmaxf(z, LEAST_T), et);
  };
#pragma unroll
  for (int u = 0; u < PART_U; ++u) {
    add(v[u].x);
    add(v[u].y);
    add(v[u].z);
    add(v[u].w);
  }
  add(v1);
  const Two both = over_block<PART_NT, Both<AddF32>>(Two{s, et}, reinterpret_cast<Two*>(lds + PART_NT / 64));
  if (t == 0) parts[row * np + part] = f4{m, both.a, both.b, 0.f};
}

// Two float4s a thread: (6288, 32000) of pairs 322 us, with one 329, with four 335; (4096, 50257) with
// entropies, both directions, 325 and with four 343.
constexpr int BWD_NT = 256, BWD_U = 2;
// Rows of fewer classes go a wave a chunk: both directions of (16384, 256) 17 us against 31, of (16384,
// 2051) 76 against 91.
constexpr int BWD_SHORT = 4096;

// A unit of TPU threads (a block, or a wave in rows of few classes) takes a chunk of a row.
template <int TPU, bool ENT, bool NTS>
__global__ __launch_bounds__(BWD_NT) void token_bwd_k(const float* __restrict__ x, const int64_t* __restrict__ ids,
                                                      const float* __restrict__ saved, const float* __restrict__ gl,
                                                      const float* __restrict__ gh, const float* __restrict__ gloss,
                                                      float* __restrict__ dx, int c, int chunks, int64_t row0, unsigned rows,
                                                      float scale2, float inv_t, int* guard, const MeanOf mean) {
  static_assert(BWD_NT == MEAN_NT);  // the block more that takes a mean
  const unsigned more = mean.count ? 1 : 0;
  if (blockIdx.x < more) {
    mean.by_block();
    return;
  }
  // the last rows first: the Infinity Cache still has some of what the forward read last
  const unsigned unit = (blockIdx.x - more) * (BWD_NT / TPU) + threadIdx.x / TPU;
  if (unit >= rows * (unsigned)chunks) return;
  const RowPiece of = TPU == BWD_NT ? RowPiece(unit, rows, (unsigned)chunks) : RowPiece(unit, 0, (unsigned)chunks);
  const int64_t row = row0 + rows - 1 - of.row;
  const int chunk = of.piece;
  const int t = threadIdx.x & (TPU - 1);
  const int64_t id = ids[row];
  const f4 sv = *reinterpret_cast<const f4u*>(saved + 4 * row);
  const float up = (gloss ? gloss[0] : 1.f) * inv_t;
  // a gradient of 0 stays 0 under an upstream that is not finite too
  auto times = [&](float g) { return g == 0.f ? 0.f : g * up; };
  const float a = gl ? times(gl[row]) : 0.f, b = ENT ? times(gh[row]) : 0.f;
  if (id >= c && t == 0) atomicOr(guard, 1);
  const bool none = id < 0 || id >= c || (a == 0.f && b == 0.f);
  const float* xr = x + row * c;
  float* dr = dx + row * c;
  // the float4s as the logits lie; the gradient may lie otherwise
  const RowLay<> lay(xr, c);
  const f4* x4 = reinterpret_cast<const f4*>(xr + lay.head);
  f4u* d4 = reinterpret_cast<f4u*>(dr + lay.head);
  auto put = [&](const f4& v, int q) {
    if constexpr (NTS) __builtin_nontemporal_store(v, d4 + q);
    else d4[q] = v;
  };
  // a wave's chunks are as long as each other, in lines of 128 bytes
  const int each = TPU == BWD_NT ? TPU * BWD_U : ((lay.c4 + chunks - 1) / chunks + 7) & ~7;
  const int c0 = chunk * each + t, end = min(chunk * each + each, lay.c4);
  const int e = chunk == 0 ? lay.edge(t, c) : -1;
  if (none) {
#pragma unroll
    for (int u = 0; u < BWD_U; ++u)
      if (c0 + u * TPU < end) put(f4{0.f, 0.f, 0.f, 0.f}, c0 + u * TPU);
    if (e >= 0) dr[e] = 0.f;
    return;
  }
  f4 v[BWD_U];
#pragma unroll
  for (int u = 0; u < BWD_U; ++u) {
    const int q = c0 + u * TPU;
    if (q < end) v[u] = ld_stream(x4 + q);
  }
  const float m = sv.x, rest = sv.y, total = sv.z, off = sv.w;
  const float alpha = -(a + b * off) / total, beta = -b * (float)LOG_2 / total;
  auto grad = [&](float xv) {
    const float z = (xv - m) * scale2;
    const float p = __builtin_amdgcn_exp2f(z);
    return ENT ? p * fmaf(beta, fmaxf(z, LEAST_T), alpha) : p * alpha;
  };
  auto chosen = [&](float xv) {
    const float z = (xv - m) * scale2;
    const float q = __builtin_amdgcn_exp2f(z) / total;
    return a * (rest / total) - (ENT ? b * q * fmaf((float)LOG_2, fmaxf(z, LEAST_T), off) : 0.f);
  };
  const int at = lay.slot((int)id), comp = lay.component((int)id);
#pragma unroll
  for (int u = 0; u < BWD_U; ++u) {
    const int q = c0 + u * TPU;
    if (q >= end) continue;
    f4 d = f4{grad(v[u].x), grad(v[u].y), grad(v[u].z), grad(v[u].w)};
    if (q == at) d = put_at(d, comp, chosen(xr[id]));
    put(d, q);
  }
  if (e >= 0) dr[e] = e == (int)id ? chosen(xr[e]) : grad(xr[e]);
}

struct LogpOp {
  static constexpr bool SUMMED = true;
  static constexpr bool SAME_BITS = false;  // there is one way
  float *logp, *entropy, *saved;
  struct Given {};
  __device__ __forceinline__ Given load(int64_t) const { return {}; }
  __device__ __forceinline__ Two finish(int64_t row, const Given&, const RowStats& r, bool lead) const {
    if (!lead) return {0.f, 0.f};
    logp[row] = (float)r.logp;
    if (entropy) entropy[row] = (float)r.entropy;
    if (saved) save_row(saved, row, r);
    return {0.f, 0.f};
  }
  __device__ __forceinline__ void skip(int64_t row) const {
    logp[row] = 0.f;
    if (entropy) entropy[row] = 0.f;
    if (saved) save_nothing(saved, row);
  }
};

}  // namespace

namespace {
__global__ __launch_bounds__(256) void zero_words_k(uint64_t* __restrict__ p, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) p[i] = 0;
}
}  // namespace

Cluster start_cluster(void* at, int64_t n, int blocks) {
  const int64_t words = cluster_bytes(n, blocks) / (int64_t)sizeof(uint64_t);
  zero_words_k<<<dim3((unsigned)ceil_div(words, 256)), dim3(256), 0, stream()>>>(static_cast<uint64_t*>(at), words);
  // polls of about 1 us: a wait past some seconds is a failure (never seen); OXI_CLUSTER_SPIN_LIMIT=-1 fails
  // every wait, to test that path
  const char* sl = std::getenv("OXI_CLUSTER_SPIN_LIMIT");
  const int spin_limit = sl && std::strcmp(sl, "-1") == 0 ? -1 : 1 << 22;
  return {static_cast<uint64_t*>(at) + 8, static_cast<uint32_t*>(at), blocks, spin_limit};
}

int check_token_rows(const char* what, int64_t n, int64_t c, float temperature) {
  if (n < 0 || c < 0) return fail(OXI_INVALID_ARGUMENT, "%s: negative size", what);
  if (c > ((int64_t)1 << 30) || !grid_fits(n, 1024))
    return fail(OXI_INVALID_ARGUMENT, "%s: size exceeds the kernel limits", what);
  if (!(temperature > 0.f) || std::isinf(temperature))
    return fail(OXI_INVALID_ARGUMENT, "%s: the temperature must be positive, got %g", what, (double)temperature);
  if (std::isinf((float)(1.4426950408889634 / temperature)))  // the kernels' factor of the logits
    return fail(OXI_INVALID_ARGUMENT, "%s: a temperature of %g has no 32-bit reciprocal", what, (double)temperature);
  if (n && c == 0) return fail(OXI_INVALID_ARGUMENT, "%s: zero classes", what);
  return OXI_OK;
}

TokenRows token_rows(const float* x, const int64_t* ids, int64_t n, int64_t c, float temperature) {
  TokenRows in{};
  in.x = x;
  in.ids = ids;
  in.n = n;
  in.c = (int)c;
  in.scale2 = (float)(1.4426950408889634 / temperature);
  in.inv_t = 1.0 / (double)temperature;
  in.skew = (double)in.scale2 * (LOG_2 * (double)temperature) - 1.0;
  in.guard = guard_flag();
  return in;
}

// Rows that one launch of `blocks` blocks a row takes.
// (a block less than a launch may have: the backward's may have one more)
static int64_t rows_a_launch(int64_t blocks, int threads) { return (0xffffffffll / threads - 1) / blocks; }

int launch_token_parts(const TokenRows& in, f4* parts, const char* what) {
  const int64_t np = row_parts(in.c), most = rows_a_launch(np, PART_NT);
  for (int64_t r0 = 0; r0 < in.n; r0 += most) {
    const int64_t rows = in.n - r0 < most ? in.n - r0 : most;
    token_part_k<<<dim3((unsigned)(rows * np)), dim3(PART_NT), 0, stream()>>>(in, parts, (int)np, r0);
  }
  return check_launch(what);
}

int launch_token_bwd(const float* x, const int64_t* ids, const float* saved, const float* gl, const float* gh,
                     const float* gloss, float* dx, int64_t n, int64_t c, float temperature, const char* what,
                     const MeanOf& mean) {
  const bool waves = c < BWD_SHORT;
  const int64_t chunks = ceil_div(c, (int64_t)(waves ? 64 : BWD_NT) * BWD_U * 4), most = rows_a_launch(chunks, BWD_NT);
  const float scale2 = (float)(1.4426950408889634 / temperature), inv_t = (float)(1.0 / (double)temperature);
  const bool nt = nt_stream_stores(n * c * 4);
  for (int64_t r0 = 0; r0 < n; r0 += most) {
    const int64_t rows = n - r0 < most ? n - r0 : most;
    const MeanOf also = r0 ? MeanOf{} : mean;
    const dim3 grid((unsigned)(ceil_div(rows * chunks, waves ? BWD_NT / 64 : 1) + (also.count ? 1 : 0)));
#define OXI_TB(TPU, ENT, NTS)                                                                                         \
  token_bwd_k<TPU, ENT, NTS><<<grid, dim3(BWD_NT), 0, stream()>>>(x, ids, saved, gl, gh, gloss, dx, (int)c, (int)chunks, \
                                                                  r0, (unsigned)rows, scale2, inv_t, guard_flag(), also)
#define OXI_TU(TPU)                     \
  if (gh && nt) OXI_TB(TPU, true, true); \
  else if (gh) OXI_TB(TPU, true, false); \
  else if (nt) OXI_TB(TPU, false, true); \
  else OXI_TB(TPU, false, false)
    if (waves) {
      OXI_TU(64);
    } else {
      OXI_TU(BWD_NT);
    }
#undef OXI_TU
#undef OXI_TB
  }
  return check_launch(what);
}

}  // namespace oxi

using namespace oxi;

extern "C" {

int oxi_token_logp_workspace(int64_t n, int64_t c, int64_t* bytes) {
  if (!bytes) return fail(OXI_INVALID_ARGUMENT, "token_logp_workspace: NULL result");
  if (int rc = check_token_rows("token_logp_workspace", n, c, 1.f)) return rc;
  *bytes = token_parts_bytes(n, c);
  return OXI_OK;
}

int oxi_token_logp_fwd(const float* logits, const int64_t* ids, float* logp, float* entropy, float* saved,
                       void* workspace, int64_t n, int64_t c, float temperature) {
  const char* what = "token_logp_fwd";
  if (int rc = check_token_rows(what, n, c, temperature)) return rc;
  if (n && (!logits || !ids || !logp)) return fail(OXI_INVALID_ARGUMENT, "%s: NULL tensor pointer", what);
  if (reinterpret_cast<uintptr_t>(workspace) & 15)
    return fail(OXI_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", what);
  OXI_CHECK_INIT();
  if (n == 0) return OXI_OK;
  Workspace own(workspace ? 0 : (size_t)token_parts_bytes(n, c));
  if (!workspace && !own.p) return fail_alloc(what);
  f4* parts = static_cast<f4*>(workspace ? workspace : own.p);
  return token_rows_read(token_rows(logits, ids, n, c, temperature), parts, LogpOp{logp, entropy, saved}, what);
}

int oxi_token_logp_bwd(const float* logits, const int64_t* ids, const float* saved, const float* glogp,
                       const float* gentropy, const float* gloss, float* dlogits, int64_t n, int64_t c,
                       float temperature) {
  const char* what = "token_logp_bwd";
  if (int rc = check_token_rows(what, n, c, temperature)) return rc;
  if (n && (!logits || !ids || !saved || !dlogits || (!glogp && !gentropy)))
    return fail(OXI_INVALID_ARGUMENT, "%s: NULL tensor pointer", what);
  if (n && dlogits == logits) return fail(OXI_INVALID_ARGUMENT, "%s: dlogits must not be the logits", what);
  OXI_CHECK_INIT();
  if (n == 0) return OXI_OK;
  return launch_token_bwd(logits, ids, saved, glogp, gentropy, gloss, dlogits, n, c, temperature, what);
}

}  // extern "C"

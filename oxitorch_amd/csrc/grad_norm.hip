// The joint norm of many gradient tensors and their clipping by it:
//
//   total = (sum |g|^p)^(1/p), p = 1 or 2, or max |g|
//   out = g * min(1, max_norm / (total + 1e-6))
//
// Every tensor is cut into chunks of CHUNK floats, a block each; the tensors' places
// travel in the kernel arguments, up to MOST_SLICES a launch. The terms are squared and
// summed in 64 bits (no overflow, and a sum over 10^9 terms keeps its digits), a sum a
// chunk, then one block adds the chunks' in a fixed order. The clipping reads total on
// the device, so nothing waits for the host between the two.
#include <cmath>

#include "internal.h"
#include "launch_limits.h"
#include "row64.h"
#include "rowtile.h"

namespace oxi {
namespace {

constexpr int NT = 256;
constexpr int UNROLL = 4;               // float4s in flight a thread
constexpr int CHUNK = NT * UNROLL * 4;  // floats
constexpr int MOST_SLICES = 96;

struct Slices {
  const float* g[MOST_SLICES];
  float* out[MOST_SLICES];
  int64_t n[MOST_SLICES];
  uint32_t end[MOST_SLICES];  // blocks up to and with slice s
  int count;
};

__device__ __forceinline__ int slice_of(const Slices& a, uint32_t b) {
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (b < a.end[mid]) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// KIND 0: max, 1: sum, 2: sum of squares. parts[first + block] = the chunk's.
template <int KIND>
__global__ __launch_bounds__(NT) void norm_part_k(const Slices a, double* __restrict__ parts, int64_t first) {
  __shared__ double red[NT / 64];
  const int s = slice_of(a, blockIdx.x);
  const int64_t n = a.n[s];
  const int64_t e0 = (int64_t)(blockIdx.x - (s ? a.end[s - 1] : 0u)) * CHUNK;
  const float* g = a.g[s];
  double acc = KIND == 0 ? (double)NEG_INF : 0.0;
  auto add = [&](float v) {
    if constexpr (KIND == 0) acc = fmax(acc, (double)fabsf(v));  // a NaN is passed over
    else if constexpr (KIND == 1) acc += (double)fabsf(v);
    else acc = fma((double)v, (double)v, acc);
  };
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const int64_t e = e0 + (int64_t)(u * NT + threadIdx.x) * 4;
    if (e + 4 <= n) {
      const f4 v = *reinterpret_cast<const f4u*>(g + e);
      add(v.x);
      add(v.y);
      add(v.z);
      add(v.w);
    } else {
      for (int64_t i = e; i < n; ++i) add(g[i]);
    }
  }
  if constexpr (KIND == 0) {
    acc = (double)over_block<NT, MaxF32>((float)acc, reinterpret_cast<float*>(red));
  } else {
    acc = over_block<NT, AddF64>(acc, red);
  }
  if (threadIdx.x == 0) parts[first + blockIdx.x] = acc;
}

template <int KIND>
__global__ __launch_bounds__(1024) void norm_total_k(const double* __restrict__ parts, int64_t n,
                                                     double* __restrict__ total) {
  __shared__ double red[1024 / 64];
  double acc = KIND == 0 ? (double)NEG_INF : 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) acc = KIND == 0 ? fmax(acc, parts[i]) : acc + parts[i];
  if constexpr (KIND == 0) acc = (double)over_block<1024, MaxF32>((float)acc, reinterpret_cast<float*>(red));
  else acc = over_block<1024, AddF64>(acc, red);
  if (threadIdx.x == 0) total[0] = KIND == 2 ? sqrt(acc) : acc;
}

__global__ __launch_bounds__(NT) void clip_k(const Slices a, const double* __restrict__ total, double max_norm) {
  const int s = slice_of(a, blockIdx.x);
  const int64_t n = a.n[s];
  const int64_t e0 = (int64_t)(blockIdx.x - (s ? a.end[s - 1] : 0u)) * CHUNK;
  const float* g = a.g[s];
  float* out = a.out[s];
  const double ratio = max_norm / (total[0] + 1e-6);
  const bool clip = ratio < 1.0;  // not for a NaN
  if (!clip && out == g) return;
  const float k = clip ? (float)ratio : 1.f;
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const int64_t e = e0 + (int64_t)(u * NT + threadIdx.x) * 4;
    if (e + 4 <= n) {
      const f4 v = *reinterpret_cast<const f4u*>(g + e);
      *reinterpret_cast<f4u*>(out + e) = v * k;
    } else {
      for (int64_t i = e; i < n; ++i) out[i] = g[i] * k;
    }
  }
}

int check_slices(const char* what, const oxi_grad_slice* slices, int count, bool outs, int64_t* chunks) {
  if (count < 0) return fail(OXI_INVALID_ARGUMENT, "%s: negative slice count", what);
  if (count > 0 && !slices) return fail(OXI_INVALID_ARGUMENT, "%s: NULL slice array", what);
  *chunks = 0;
  for (int i = 0; i < count; ++i) {
    if (slices[i].n < 0) return fail(OXI_INVALID_ARGUMENT, "%s: slice %d has a negative size", what, i);
    if (slices[i].n == 0) continue;
    if (!slices[i].g || (outs && !slices[i].out))
      return fail(OXI_INVALID_ARGUMENT, "%s: slice %d has a NULL pointer", what, i);
    if (slices[i].n > INT64_MAX - CHUNK || !grid_fits(ceil_div(slices[i].n, CHUNK), NT))
      return fail(OXI_INVALID_ARGUMENT, "%s: slice %d is too large", what, i);
    *chunks += ceil_div(slices[i].n, CHUNK);
  }
  return OXI_OK;
}

// Calls launch(slices, blocks, blocks before) for as many slices at once as fit.
template <class F>
int for_slices(const oxi_grad_slice* slices, int count, const char* what, F launch) {
  Slices a{};
  int64_t blocks = 0, before = 0;
  int rc = OXI_OK;
  auto flush = [&]() {
    if (!a.count) return;
    launch(a, (unsigned)blocks, before);
    if (rc == OXI_OK) rc = check_launch(what);
    before += blocks;
    blocks = 0;
    a.count = 0;
  };
  for (int i = 0; i < count; ++i) {
    if (slices[i].n == 0) continue;
    const int64_t nb = ceil_div(slices[i].n, CHUNK);
    if (a.count == MOST_SLICES || !grid_fits(blocks + nb, NT)) flush();
    a.g[a.count] = slices[i].g;
    a.out[a.count] = slices[i].out;
    a.n[a.count] = slices[i].n;
    blocks += nb;
    a.end[a.count++] = (uint32_t)blocks;
  }
  flush();
  return rc;
}

}  // namespace
}  // namespace oxi

using namespace oxi;

extern "C" {

int oxi_grad_norm_workspace(const oxi_grad_slice* slices, int count, int64_t* bytes) {
  if (!bytes) return fail(OXI_INVALID_ARGUMENT, "grad_norm_workspace: NULL result");
  int64_t chunks = 0;
  if (int rc = check_slices("grad_norm_workspace", slices, count, false, &chunks)) return rc;
  *bytes = chunks * (int64_t)sizeof(double);
  return OXI_OK;
}

int oxi_grad_norm(const oxi_grad_slice* slices, int count, double norm_type, double* total, void* workspace) {
  const char* what = "grad_norm";
  int64_t chunks = 0;
  if (int rc = check_slices(what, slices, count, false, &chunks)) return rc;
  const int kind = norm_type == 2.0 ? 2 : norm_type == 1.0 ? 1 : std::isinf(norm_type) && norm_type > 0 ? 0 : -1;
  if (kind < 0) return fail(OXI_INVALID_ARGUMENT, "%s: the norm must be 1, 2 or infinite, got %g", what, norm_type);
  if (!total) return fail(OXI_INVALID_ARGUMENT, "%s: total must not be NULL", what);
  if ((reinterpret_cast<uintptr_t>(total) | reinterpret_cast<uintptr_t>(workspace)) & 7)
    return fail(OXI_INVALID_ARGUMENT, "%s: total and the workspace must be 8-byte aligned", what);
  OXI_CHECK_INIT();
  Workspace own(workspace ? 0 : (size_t)chunks * sizeof(double));
  if (chunks && !workspace && !own.p) return fail_alloc(what);
  double* parts = static_cast<double*>(workspace ? workspace : own.p);
  const int rc = for_slices(slices, count, what, [&](const Slices& a, unsigned blocks, int64_t before) {
    if (kind == 0) norm_part_k<0><<<blocks, NT, 0, stream()>>>(a, parts, before);
    else if (kind == 1) norm_part_k<1><<<blocks, NT, 0, stream()>>>(a, parts, before);
    else norm_part_k<2><<<blocks, NT, 0, stream()>>>(a, parts, before);
  });
  if (rc) return rc;
  if (kind == 0) norm_total_k<0><<<1, 1024, 0, stream()>>>(parts, chunks, total);
  else if (kind == 1) norm_total_k<1><<<1, 1024, 0, stream()>>>(parts, chunks, total);
  else norm_total_k<2><<<1, 1024, 0, stream()>>>(parts, chunks, total);
  return check_launch(what);
}

int oxi_grad_clip(const oxi_grad_slice* slices, int count, const double* total, double max_norm) {
  const char* what = "grad_clip";
  int64_t chunks = 0;
  if (int rc = check_slices(what, slices, count, true, &chunks)) return rc;
  if (!total) return fail(OXI_INVALID_ARGUMENT, "%s: total must not be NULL", what);
  if (reinterpret_cast<uintptr_t>(total) & 7)
    return fail(OXI_INVALID_ARGUMENT, "%s: total must be 8-byte aligned", what);
  if (std::isnan(max_norm)) return fail(OXI_INVALID_ARGUMENT, "%s: max_norm is NaN", what);
  OXI_CHECK_INIT();
  return for_slices(slices, count, what, [&](const Slices& a, unsigned blocks, int64_t) {
    clip_k<<<blocks, NT, 0, stream()>>>(a, total, max_norm);
  });
}

}  // extern "C"

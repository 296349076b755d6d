// The joint norm of many gradient tensors and their clipping by it:
//
//   total = (sum |g|^p)^(1/p), p = 1 or 2, or max |g|
//   out = g * min(1, max_norm / (total + 1e-6))
//
// Every tensor is cut into chunks, a block each; the tensors' places travel in the kernel
// arguments, up to MOST_SLICES a launch, and one that passes a launch is cut (grad_slices.h). The terms are squared and summed in 64 bits (no
// overflow, and a sum over 10^9 terms keeps its digits), a sum a chunk, then one block
// adds the chunks' in a fixed order. The clipping reads total on the device, so nothing
// waits for the host between the two.
//
// HBM bounds it: 354 M floats in 242 tensors, the norm's parts 223 us (6.3 TB/s) and clipping 445 (6.4);
// both calls 668 us into other tensors, 705 in place.
#include <cmath>

#include "grad_slices.h"
#include "internal.h"
#include "launch_limits.h"
#include "row64.h"
#include "rowtile.h"

namespace oxi {
namespace {

constexpr int NT = 256;
constexpr int UNROLL = 4;               // float4s in flight a thread
constexpr int STEP = NT * UNROLL * 4;   // floats that a block has in flight
// Floats a block of the norm's: STEP, or, from MANY floats on, several of them, so that the
// chunks' sums are few (10^8 floats 71 us against 75, 4 * 10^7 32 against 34; with 4 steps 72 and 36).
constexpr int LONG_STEPS = 8;
constexpr int64_t MANY = (int64_t)1 << 25;
inline int64_t chunk_of(int64_t total) { return total >= MANY ? (int64_t)STEP * LONG_STEPS : STEP; }
// Of the clipping's, without a loop, whose loads would wait behind the stores before them: two float4s
// a thread (354 M floats, norm and clipping 673 us; one 682, four 675, in a loop of 8 784).
constexpr int CLIP_UNROLL = 2, CLIP_CHUNK = NT * CLIP_UNROLL * 4;
constexpr int MOST_SLICES = 96;
// What of the gradients the clipping, which begins at their end, finds in the 256 MB Infinity Cache:
// the norm loads it with plain loads (1.4 GB 675 us both together, 684 without; 165 MB 84.6 and 88.3).
constexpr int64_t REREAD_BYTES = (int64_t)208 << 20;

struct Slices {
  const float* g[MOST_SLICES];
  float* out[MOST_SLICES];
  int64_t n[MOST_SLICES];
  uint32_t end[MOST_SLICES];  // blocks up to and with slice s
  int count;
  int64_t chunk;
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
// AGAIN: plain loads, for what the clipping then finds in the Infinity Cache.
template <int KIND, bool AGAIN>
__global__ __launch_bounds__(NT) void norm_part_k(const Slices a, double* __restrict__ parts, int64_t first) {
  __shared__ double red[NT / 64];
  const int s = slice_of(a, blockIdx.x);
  int64_t e0 = (int64_t)(blockIdx.x - (s ? a.end[s - 1] : 0u)) * a.chunk;
  const int64_t n = min(a.n[s], e0 + a.chunk);
  const float* g = a.g[s];
  double acc = KIND == 0 ? (double)NEG_INF : 0.0;
  auto add = [&](float v) {
    if constexpr (KIND == 0) acc = fmax(acc, (double)fabsf(v));  // a NaN is passed over
    else if constexpr (KIND == 1) acc += (double)fabsf(v);
    else acc = fma((double)v, (double)v, acc);
  };
  for (; e0 + STEP <= n; e0 += STEP) {
    f4 v[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const f4u* p = reinterpret_cast<const f4u*>(g + e0) + u * NT + threadIdx.x;
      if constexpr (AGAIN) v[u] = *p;
      else v[u] = __builtin_nontemporal_load(p);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      add(v[u].x);
      add(v[u].y);
      add(v[u].z);
      add(v[u].w);
    }
  }
  for (int64_t e = e0 + threadIdx.x; e < n; e += NT) add(g[e]);
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

// The launch takes its slices in turn, each from its end; the launches go from the last slices, where the
// norm's pass has just been.
template <bool NTS>
__global__ __launch_bounds__(NT) void clip_k(const Slices a, const double* __restrict__ total, double max_norm) {
  const uint32_t b = gridDim.x - 1 - blockIdx.x;
  const int s = slice_of(a, b);
  const int64_t e0 = (int64_t)(b - (s ? a.end[s - 1] : 0u)) * CLIP_CHUNK;
  const int64_t n = min(a.n[s], e0 + CLIP_CHUNK);
  const float* g = a.g[s];
  float* out = a.out[s];
  const bool whole = n - e0 == CLIP_CHUNK;
  f4 v[CLIP_UNROLL];
  auto load = [&]() {
#pragma unroll
    for (int u = 0; u < CLIP_UNROLL; ++u)
      v[u] = __builtin_nontemporal_load(reinterpret_cast<const f4u*>(g + e0) + u * NT + threadIdx.x);
  };
  // into another tensor the gradients are read in any case: before the norm is known
  // (354 M floats, both together 668 us; behind it 676)
  if (whole && out != g) load();
  const double ratio = max_norm / (total[0] + 1e-6);
  const bool clip = ratio < 1.0;  // not for a NaN
  if (!clip && out == g) return;
  const float k = clip ? (float)ratio : 1.f;
  if (!whole) {
    for (int64_t e = e0 + threadIdx.x; e < n; e += NT) out[e] = g[e] * k;
    return;
  }
  if (out == g) load();
#pragma unroll
  for (int u = 0; u < CLIP_UNROLL; ++u) {
    f4u* p = reinterpret_cast<f4u*>(out + e0) + u * NT + threadIdx.x;
    if constexpr (NTS) __builtin_nontemporal_store(v[u] * k, p);
    else *p = v[u] * k;
  }
}

int check_slices(const char* what, const oxi_grad_slice* slices, int count, bool outs, int64_t* total) {
  if (count < 0) return fail(OXI_INVALID_ARGUMENT, "%s: negative slice count", what);
  if (count > 0 && !slices) return fail(OXI_INVALID_ARGUMENT, "%s: NULL slice array", what);
  *total = 0;
  for (int i = 0; i < count; ++i) {
    if (slices[i].n < 0) return fail(OXI_INVALID_ARGUMENT, "%s: slice %d has a negative size", what, i);
    if (slices[i].n == 0) continue;
    if (!slices[i].g || (outs && !slices[i].out))
      return fail(OXI_INVALID_ARGUMENT, "%s: slice %d has a NULL pointer", what, i);
    if (slices[i].n > ((int64_t)1 << 40)) return fail(OXI_INVALID_ARGUMENT, "%s: slice %d is too large", what, i);
    *total += slices[i].n;
  }
  return OXI_OK;
}

// Chunks of all slices, which hold `total` floats.
int64_t chunks_of(const oxi_grad_slice* slices, int count, int64_t total) {
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) chunks += ceil_div(slices[i].n, chunk_of(total));
  return chunks;
}

// Calls launch(slices, blocks, blocks before) for as many slices at once as fit (grad_slices.h), in
// order or from the last on.
template <class F>
int for_slices(const oxi_grad_slice* slices, int count, int64_t chunk, bool back, const char* what, F launch) {
  Slices a{};
  a.chunk = chunk;
  int64_t blocks = 0, before = 0;
  int rc = OXI_OK;
  walk_slices(
      [&](int i) { return slices[i].n; }, count, chunk, NT, MOST_SLICES, back,
      [&](int i, int64_t e0, int64_t n, int64_t nb) {
        a.g[a.count] = slices[i].g + e0;
        a.out[a.count] = slices[i].out ? slices[i].out + e0 : nullptr;
        a.n[a.count] = n;
        blocks += nb;
        a.end[a.count++] = (uint32_t)blocks;
      },
      [&]() {
        launch(a, (unsigned)blocks, before);
        if (rc == OXI_OK) rc = check_launch(what);
        before += blocks;
        blocks = 0;
        a.count = 0;
      });
  return rc;
}

}  // namespace
}  // namespace oxi

using namespace oxi;

extern "C" {

int oxi_grad_norm_workspace(const oxi_grad_slice* slices, int count, int64_t* bytes) {
  if (!bytes) return fail(OXI_INVALID_ARGUMENT, "grad_norm_workspace: NULL result");
  int64_t n = 0;
  if (int rc = check_slices("grad_norm_workspace", slices, count, false, &n)) return rc;
  *bytes = chunks_of(slices, count, n) * (int64_t)sizeof(double);
  return OXI_OK;
}

int oxi_grad_norm(const oxi_grad_slice* slices, int count, double norm_type, double* total, void* workspace) {
  const char* what = "grad_norm";
  int64_t n = 0;
  if (int rc = check_slices(what, slices, count, false, &n)) return rc;
  const int kind = norm_type == 2.0 ? 2 : norm_type == 1.0 ? 1 : std::isinf(norm_type) && norm_type > 0 ? 0 : -1;
  if (kind < 0) return fail(OXI_INVALID_ARGUMENT, "%s: the norm must be 1, 2 or infinite, got %g", what, norm_type);
  if (!total) return fail(OXI_INVALID_ARGUMENT, "%s: total must not be NULL", what);
  if ((reinterpret_cast<uintptr_t>(total) | reinterpret_cast<uintptr_t>(workspace)) & 7)
    return fail(OXI_INVALID_ARGUMENT, "%s: total and the workspace must be 8-byte aligned", what);
  OXI_CHECK_INIT();
  const int64_t chunks = chunks_of(slices, count, n);
  Workspace own(workspace ? 0 : (size_t)chunks * sizeof(double));
  if (chunks && !workspace && !own.p) return fail_alloc(what);
  double* parts = static_cast<double*>(workspace ? workspace : own.p);
  // launches that hold some of the last chunks, with which the clipping begins, read with plain loads
  const int64_t hot = chunks - REREAD_BYTES / (4 * chunk_of(n));
  const int rc = for_slices(slices, count, chunk_of(n), false, what, [&](const Slices& a, unsigned blocks, int64_t before) {
    const bool again = before + blocks > hot;
#define OXI_NP(KIND)                                                                        \
  if (again) norm_part_k<KIND, true><<<blocks, NT, 0, stream()>>>(a, parts, before);        \
  else norm_part_k<KIND, false><<<blocks, NT, 0, stream()>>>(a, parts, before)
    if (kind == 0) {
      OXI_NP(0);
    } else if (kind == 1) {
      OXI_NP(1);
    } else {
      OXI_NP(2);
    }
#undef OXI_NP
  });
  if (rc) return rc;
  if (kind == 0) norm_total_k<0><<<1, 1024, 0, stream()>>>(parts, chunks, total);
  else if (kind == 1) norm_total_k<1><<<1, 1024, 0, stream()>>>(parts, chunks, total);
  else norm_total_k<2><<<1, 1024, 0, stream()>>>(parts, chunks, total);
  return check_launch(what);
}

int oxi_grad_clip(const oxi_grad_slice* slices, int count, const double* total, double max_norm) {
  const char* what = "grad_clip";
  int64_t n = 0;
  if (int rc = check_slices(what, slices, count, true, &n)) return rc;
  if (!total) return fail(OXI_INVALID_ARGUMENT, "%s: total must not be NULL", what);
  if (reinterpret_cast<uintptr_t>(total) & 7)
    return fail(OXI_INVALID_ARGUMENT, "%s: total must be 8-byte aligned", what);
  if (std::isnan(max_norm)) return fail(OXI_INVALID_ARGUMENT, "%s: max_norm is NaN", what);
  OXI_CHECK_INIT();
  const bool nt = nt_stream_stores(n * 4);
  return for_slices(slices, count, CLIP_CHUNK, true, what, [&](const Slices& a, unsigned blocks, int64_t) {
    if (nt) clip_k<true><<<blocks, NT, 0, stream()>>>(a, total, max_norm);
    else clip_k<false><<<blocks, NT, 0, stream()>>>(a, total, max_norm);
  });
}

}  // extern "C"

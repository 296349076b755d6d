// RMS norm of a residual sum for gfx950: h = x + r and y = rms_norm(h) in one
// pass, its VJP with the residual stream's own gradient added, and the forward
// with y in 8-bit floating point with a scale per group of columns.
//
//   h = x + r,  inv = 1/sqrt(sum(h*h)/H + eps),  y = (h*inv)*w
//   dx = gh + d, dw = sum over rows of gy*xh,  xh = h*inv, gw = gy*w
//   d = gw*inv (the inverse held constant) or (gw - xh*mean(gw*xh))*inv
//   e4m3: s = max(max|y|/448, 2^-126) over a group, q = e4m3(y/s)
//
// A row crosses HBM once a kernel: the forward moves 16 bytes an element (reads x
// and r, writes h and y) where an add and a norm move 20, the VJP 16 (h, gy, gh,
// dx) where the norm's VJP and an add move 24, the 8-bit forward 13.
#include <algorithm>

#include "norm_bwd_impl.h"

namespace oxi {
namespace {

constexpr float E4M3_MAX = 448.0f;

// max(amax/448, 2^-126): a group of zeros (or of NaN) gets a scale that can
// still be divided by.
__device__ __forceinline__ float e4m3_scale(float amax) { return fmaxf(amax / E4M3_MAX, 0x1p-126f); }

// The code of y / s (gfx950 converts to OCP e4m3, to nearest even). The quotient
// is at most 448 but for its rounding; a NaN passes the clamp and gets its code.
__device__ __forceinline__ float e4m3_ready(float y, float s) {
  const float v = y / s;
  return v != v ? v : __builtin_amdgcn_fmed3f(v, -E4M3_MAX, E4M3_MAX);
}
__device__ __forceinline__ uint32_t e4m3_pack(f4 v) {
  int p = __builtin_amdgcn_cvt_pk_fp8_f32(v.x, v.y, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v.z, v.w, p, true);
}
__device__ __forceinline__ uint8_t e4m3_code(float v) {
  return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 0xff);
}

// ---------------------------------------------------------------------------
// Rows that the register kernels do not take (fewer than 4 floats, or more than
// they hold): a block a row, which it walks twice.

// h may be x or r, so neither is restricted; a thread reads back only the h
// that it wrote.
__global__ __launch_bounds__(BS) void add_norm_fwd_loop_k(const float* x, const float* r, const float* __restrict__ w,
                                                          float* h, float* __restrict__ y, float* __restrict__ rstd,
                                                          int64_t rows, int H, float eps) {
  __shared__ float lds[BS / 64];
  const int t = threadIdx.x;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t o = row * H;
    float ss = 0.f;
    for (int c = t; c < H; c += BS) {
      const float v = x[o + c] + r[o + c];
      h[o + c] = v;
      ss += v * v;
    }
    const float inv = 1.0f / sqrtf(rsum<BS>(ss, lds) / (float)H + eps);
    if (t == 0 && rstd) rstd[row] = inv;
    for (int c = t; c < H; c += BS) {
      const float v = h[o + c] * inv;
      y[o + c] = w ? v * w[c] : v;
    }
  }
}

__global__ __launch_bounds__(BS) void add_norm_e4m3_loop_k(const float* x, const float* r, const float* __restrict__ w,
                                                           float* h, uint8_t* __restrict__ q,
                                                           float* __restrict__ scale, int64_t rows, int H, int group,
                                                           int groups, float eps) {
  __shared__ float lds[BS / 64];
  __shared__ float lm[BS / 64];
  const int t = threadIdx.x;
  const float* src = r ? h : x;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t o = row * H;
    float ss = 0.f;
    for (int c = t; c < H; c += BS) {
      float v = x[o + c];
      if (r) {
        v = v + r[o + c];
        h[o + c] = v;
      }
      ss += v * v;
    }
    const float inv = 1.0f / sqrtf(rsum<BS>(ss, lds) / (float)H + eps);  // its barriers publish h to the block
    auto at = [&](int c) {
      const float v = src[o + c] * inv;
      return w ? v * w[c] : v;
    };
    if (groups == 1) {
      float m = 0.f;
      for (int c = t; c < H; c += BS) m = fmaxf(m, fabsf(at(c)));
      const float s = e4m3_scale(group_max<BS>(m, lm));
      if (t == 0) scale[row] = s;
      for (int c = t; c < H; c += BS) q[o + c] = e4m3_code(e4m3_ready(at(c), s));
    } else {  // a wave a group
      for (int g = t >> 6; g < groups; g += BS / 64) {
        const int c0 = g * group, c1 = min(c0 + group, H);
        float m = 0.f;
        for (int c = c0 + (t & 63); c < c1; c += 64) m = fmaxf(m, fabsf(at(c)));
        const float s = e4m3_scale(wave_max(m));
        if ((t & 63) == 0) scale[row * groups + g] = s;
        for (int c = c0 + (t & 63); c < c1; c += 64) q[o + c] = e4m3_code(e4m3_ready(at(c), s));
      }
    }
  }
}

// The VJP: the block's partial row of dw lies in global memory, its own.
// dx may be gh, so neither is restricted.
template <int MODE>
__global__ __launch_bounds__(BS) void add_norm_bwd_loop_k(const float* __restrict__ h, const float* __restrict__ w,
                                                          const float* __restrict__ rstd, const float* __restrict__ gy,
                                                          const float* gh, float* dx, float* __restrict__ part,
                                                          int64_t rows, int H) {
  __shared__ float lds[BS / 64];
  const int t = threadIdx.x;
  float* pw = part ? part + (int64_t)blockIdx.x * H : nullptr;
  if (part)
    for (int c = t; c < H; c += BS) pw[c] = 0.f;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t o = row * H;
    const float inv = rstd[row];
    float s = 0.f;
    for (int c = t; c < H; c += BS) {
      const float xh = h[o + c] * inv;
      const float gv = gy[o + c];
      if (part) pw[c] += gv * xh;
      if (MODE == OXI_NORM_VJP_EXACT) s += (w ? gv * w[c] : gv) * xh;
    }
    if (!dx) continue;
    float a = 0.f;
    if (MODE == OXI_NORM_VJP_EXACT) a = rsum<BS>(s, lds) / (float)H;
    for (int c = t; c < H; c += BS) {
      const float gv = gy[o + c];
      const float gw = w ? gv * w[c] : gv;
      const float d = MODE == OXI_NORM_VJP_REF ? gw * inv : (gw - (h[o + c] * inv) * a) * inv;
      dx[o + c] = gh ? gh[o + c] + d : d;
    }
  }
}

__global__ __launch_bounds__(BS) void e4m3_dequantize_k(const uint8_t* __restrict__ q, const float* __restrict__ scale,
                                                        float* __restrict__ y, int64_t rows, int H, int group,
                                                        int groups) {
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const int c = blockIdx.x * BS + threadIdx.x;
    if (c < H) y[row * H + c] = __builtin_amdgcn_cvt_f32_fp8(q[row * H + c], 0) * scale[row * groups + c / group];
  }
}

// ---------------------------------------------------------------------------
// Host dispatch.

int check_sizes(const char* what, int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0)
    return fail(OXI_INVALID_ARGUMENT, "%s: negative size (%lld, %lld)", what, (long long)rows, (long long)cols);
  if (cols > (int64_t)1 << 30 || rows > ((int64_t)1 << 31) - 1)
    return fail(OXI_INVALID_ARGUMENT, "%s: size (%lld, %lld) exceeds the kernel limits", what, (long long)rows,
                (long long)cols);
  return OXI_OK;
}

int check_group(const char* what, int64_t cols, int64_t group) {
  if (group != 32 && group != 64 && group != 128 && group != 256 && group != cols)
    return fail(OXI_INVALID_ARGUMENT, "%s: groups of %lld columns: 32, 64, 128, 256 or the row's %lld are taken", what,
                (long long)group, (long long)cols);
  return OXI_OK;
}

// Blocks that walk the rows in a grid stride.
int64_t walk_blocks(int64_t rows) { return std::min<int64_t>(rows, (int64_t)cu_count() * 16); }

int64_t bwd_blocks(int64_t rows) { return std::min<int64_t>(rows, cu_count()); }

}  // namespace
}  // namespace oxi

using namespace oxi;

extern "C" {

int oxi_add_rms_norm_fwd(const float* x, const float* r, const float* w, float* h, float* y, float* rstd,
                         int64_t rows, int64_t cols, float eps) {
  if (int rc = check_sizes("add_rms_norm_fwd", rows, cols)) return rc;
  if (rows == 0) return OXI_OK;
  if (cols == 0) return fail(OXI_INVALID_ARGUMENT, "add_rms_norm_fwd: cannot normalize a zero-length last dim");
  if (!x || !r || !h || !y) return fail(OXI_INVALID_ARGUMENT, "add_rms_norm_fwd: NULL tensor pointer");
  if (y == x || y == r || y == h) return fail(OXI_INVALID_ARGUMENT, "add_rms_norm_fwd: y must not be x, r or h");
  OXI_CHECK_INIT();
  add_norm_fwd_loop_k<<<dim3((unsigned)walk_blocks(rows)), dim3(BS), 0, stream()>>>(x, r, w, h, y, rstd, rows,
                                                                                   (int)cols, eps);
  return check_launch("add_rms_norm_fwd");
}

int oxi_add_rms_norm_bwd_workspace(int64_t rows, int64_t cols, int64_t* bytes) {
  if (int rc = check_sizes("add_rms_norm_bwd_workspace", rows, cols)) return rc;
  if (!bytes) return fail(OXI_INVALID_ARGUMENT, "add_rms_norm_bwd_workspace: NULL result pointer");
  OXI_CHECK_INIT();
  *bytes = rows && cols ? (int64_t)sizeof(float) * bwd_blocks(rows) * cols : 0;
  return OXI_OK;
}

int oxi_add_rms_norm_bwd(const float* h, const float* w, const float* rstd, const float* gy, const float* gh,
                         float* dx, float* dw, void* workspace, int64_t rows, int64_t cols, int mode) {
  if (int rc = check_sizes("add_rms_norm_bwd", rows, cols)) return rc;
  if (mode != OXI_NORM_VJP_REF && mode != OXI_NORM_VJP_EXACT)
    return fail(OXI_INVALID_ARGUMENT, "add_rms_norm_bwd: unknown VJP mode %d", mode);
  if (rows && cols) {
    if (!h || !rstd || !gy) return fail(OXI_INVALID_ARGUMENT, "add_rms_norm_bwd: NULL tensor pointer");
    if (dx && (dx == h || dx == gy)) return fail(OXI_INVALID_ARGUMENT, "add_rms_norm_bwd: dx must not be h or gy");
    if (reinterpret_cast<uintptr_t>(workspace) & 7u)
      return fail(OXI_INVALID_ARGUMENT, "add_rms_norm_bwd: the workspace at %p is not 8-byte aligned", workspace);
  }
  OXI_CHECK_INIT();
  if (rows == 0 || cols == 0) return dw && cols ? oxi_fill(dw, cols, 0.f) : OXI_OK;
  if (!dx && !dw) return OXI_OK;
  const int64_t nb = bwd_blocks(rows);
  Workspace ws(dw && !workspace ? sizeof(float) * (size_t)nb * (size_t)cols : 0);
  float* part = !dw ? nullptr : workspace ? static_cast<float*>(workspace) : ws.as<float>();
  if (dw && !part) return fail_alloc("add_rms_norm_bwd: column partials");
  if (mode == OXI_NORM_VJP_REF)
    add_norm_bwd_loop_k<OXI_NORM_VJP_REF><<<dim3((unsigned)nb), dim3(BS), 0, stream()>>>(h, w, rstd, gy, gh, dx, part,
                                                                                         rows, (int)cols);
  else
    add_norm_bwd_loop_k<OXI_NORM_VJP_EXACT><<<dim3((unsigned)nb), dim3(BS), 0, stream()>>>(h, w, rstd, gy, gh, dx,
                                                                                           part, rows, (int)cols);
  if (int rc = check_launch("add_rms_norm_bwd")) return rc;
  if (!dw) return OXI_OK;
  const dim3 fg((unsigned)ceil_div(cols, FIN_C), 1);
  col_finish_k<16><<<fg, dim3(FIN_C * 16), 0, stream()>>>(part, (int)nb, (int)cols, dw, nullptr);
  return check_launch("add_rms_norm_bwd: weight gradient");
}

int oxi_add_rms_norm_e4m3_fwd(const float* x, const float* r, const float* w, float* h, uint8_t* q, float* scale,
                              int64_t rows, int64_t cols, int64_t group, float eps) {
  if (int rc = check_sizes("add_rms_norm_e4m3_fwd", rows, cols)) return rc;
  if (rows == 0) return OXI_OK;
  if (cols == 0) return fail(OXI_INVALID_ARGUMENT, "add_rms_norm_e4m3_fwd: cannot normalize a zero-length last dim");
  if (int rc = check_group("add_rms_norm_e4m3_fwd", cols, group)) return rc;
  if (!x || (r && !h) || !q || !scale) return fail(OXI_INVALID_ARGUMENT, "add_rms_norm_e4m3_fwd: NULL tensor pointer");
  OXI_CHECK_INIT();
  add_norm_e4m3_loop_k<<<dim3((unsigned)walk_blocks(rows)), dim3(BS), 0, stream()>>>(
      x, r, w, h, q, scale, rows, (int)cols, (int)group, (int)ceil_div(cols, group), eps);
  return check_launch("add_rms_norm_e4m3_fwd");
}

int oxi_e4m3_dequantize(const uint8_t* q, const float* scale, float* y, int64_t rows, int64_t cols, int64_t group) {
  if (int rc = check_sizes("e4m3_dequantize", rows, cols)) return rc;
  if (rows == 0 || cols == 0) return OXI_OK;
  if (int rc = check_group("e4m3_dequantize", cols, group)) return rc;
  if (!q || !scale || !y) return fail(OXI_INVALID_ARGUMENT, "e4m3_dequantize: NULL tensor pointer");
  OXI_CHECK_INIT();
  const dim3 grid((unsigned)ceil_div(cols, BS), (unsigned)std::min<int64_t>(rows, 16384));
  e4m3_dequantize_k<<<grid, dim3(BS), 0, stream()>>>(q, scale, y, rows, (int)cols, (int)group,
                                                     (int)ceil_div(cols, group));
  return check_launch("e4m3_dequantize");
}

}  // extern "C"

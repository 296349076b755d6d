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
// Forward, a row in the registers of TPR threads.

enum { OUT_F32 = 0, OUT_E4M3 = 1 };

// Maximum over the 2^LOG lanes around this one that share lane >> LOG.
template <int LOG>
__device__ __forceinline__ float lanes_max(float v) {
  static_assert(LOG >= 3 && LOG <= 6);
  v = fmaxf(v, dpp_f32<DPP_QUAD_XOR1>(v));
  v = fmaxf(v, dpp_f32<DPP_QUAD_XOR2>(v));
  v = fmaxf(v, dpp_f32<DPP_ROW_HALF_MIRROR>(v));
  if constexpr (LOG >= 4) v = fmaxf(v, dpp_f32<DPP_ROW_MIRROR>(v));
  if constexpr (LOG >= 5) v = fmaxf(v, __shfl_xor(v, 16, 64));
  if constexpr (LOG >= 6) v = fmaxf(v, __shfl_xor(v, 32, 64));
  return v;
}

__device__ __forceinline__ float abs_max4(const f4& v) {
  return fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
}

typedef uint32_t u32u __attribute__((aligned(1)));

// An odd row's slots where the operand that they were formed from may be this
// very row: each float by the one slot that owns it. The last slot's repeated
// floats may have been read after their owner, in another wave, had written
// them: nothing is formed from them but what the owner writes.
template <int TPR, int NV>
__device__ __forceinline__ void store_owned(const RowTile<TPR, NV>& v, float* row, int H, int h4, int t) {
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = k * TPR + t;
    if (c < h4 - 1) {
      *reinterpret_cast<f4u*>(row + 4 * c) = v.v[k];
    } else if (c == h4 - 1) {
      const int e0 = H - 4;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (e0 + j >= 4 * c) row[e0 + j] = v.v[k][j];
    }
  }
}

// A block a row (four rows of at most 1024 columns), one load of each operand, one
// reduction, the stores of h issued before it. HBM bounds it: (16384, 4096) 176 us,
// 6.1 TB/s (with the VJP 348; blocks that walk their rows twice, as below, 1935);
// (8192, 4096) to e4m3 73 us, 6.0 TB/s. (8192, 1003), whose rows share cache lines,
// 24 us, 5.5 TB/s; 8 rows 3.2 us, the chain of a load, a reduction and a store.
//
// The group maxima of a row's slots: a group of 32 to 256 columns is 8 to 64
// neighbouring lanes (log_lanes), whatever the row's length; log_lanes 0 is the
// whole row. h may be x or r: every float of it is written by the thread that
// read it there (an odd row's repeated floats: see store_owned).
template <int TPR, int NV, int KIND, bool NTS, int NT, int OUT>
__global__ __launch_bounds__(NT) void add_norm_fwd_k(const float* x, const float* r, const float* __restrict__ w,
                                                     float* h, void* __restrict__ out, float* __restrict__ stat,
                                                     int64_t rows, int H_arg, float eps, int log_lanes, int groups) {
  const int H = KIND == ROW_FULL ? 4 * TPR * NV : H_arg;
  constexpr int GPB = NT / TPR;
  __shared__ float lds[2 * (NT / 64)];
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * GPB + threadIdx.x / TPR;
  if (row >= rows) return;  // GPB == 1 whenever TPR > 64: the whole block leaves together
  const int h4 = row_slots<KIND>(H);
  RowTile<TPR, NV> a, b;
  if constexpr (KIND == ROW_ODD) {
    a.load_odd(x + row * H, H, h4, t);
    if (OUT == OUT_F32 || r) b.load_odd(r + row * H, H, h4, t);
  } else {
    a.load(x + row * H, h4, t);
    if (OUT == OUT_F32 || r) b.load(r + row * H, h4, t);
  }
  if (OUT == OUT_F32 || r) {
#pragma unroll
    for (int k = 0; k < NV; ++k) a.v[k] = a.v[k] + b.v[k];
    if constexpr (KIND == ROW_ODD) store_owned(a, h + row * H, H, h4, t);
    else a.template store<NTS>(h + row * H, h4, t);
  }
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const f4 v = without_dup<KIND>(a.v[k], H, k * TPR + t);
    ss += (v.x * v.x + v.y * v.y) + (v.z * v.z + v.w * v.w);
  }
  const float inv = 1.0f / sqrtf(rsum1<TPR>(ss, lds) / (float)H + eps);
  const f4* w4 = reinterpret_cast<const f4*>(w);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = k * TPR + t;
    if (c < h4) {
      f4 o = a.v[k] * inv;
      if (w) {
        if constexpr (KIND == ROW_ODD) o = o * ld_odd(w, H, c);
        else o = o * w4[c];
      }
      a.v[k] = o;
    }
  }
  if constexpr (OUT == OUT_F32) {
    if (t == 0 && stat) stat[row] = inv;
    float* y = static_cast<float*>(out);
    if constexpr (KIND == ROW_ODD) store_owned(a, y + row * H, H, h4, t);
    else a.template store<NTS>(y + row * H, h4, t);
  } else {
    uint8_t* q = static_cast<uint8_t*>(out) + row * H;
    float* scale = stat + row * groups;
    float whole = 0.f;
    if (log_lanes == 0) {
#pragma unroll
      for (int k = 0; k < NV; ++k) whole = fmaxf(whole, abs_max4(without_dup<KIND>(a.v[k], H, k * TPR + t)));
      whole = group_max_once<TPR>(whole, lds + NT / 64);
      if (t == 0) scale[0] = e4m3_scale(whole);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = k * TPR + t;
      float m = whole;
      if (log_lanes != 0) {  // padding slots hold 0
        m = abs_max4(without_dup<KIND>(a.v[k], H, c));
        switch (log_lanes) {
          case 3: m = lanes_max<3>(m); break;
          case 4: m = lanes_max<4>(m); break;
          case 5: m = lanes_max<5>(m); break;
          default: m = lanes_max<6>(m);
        }
      }
      const float s = e4m3_scale(m);
      if (c < h4) {
        if (log_lanes != 0 && (c & ((1 << log_lanes) - 1)) == 0) scale[c >> log_lanes] = s;
        const f4 v = a.v[k];
        const uint32_t p = e4m3_pack(f4{e4m3_ready(v.x, s), e4m3_ready(v.y, s), e4m3_ready(v.z, s), e4m3_ready(v.w, s)});
        if constexpr (KIND == ROW_ODD) {
          if (c < h4 - 1) {
            *reinterpret_cast<u32u*>(q + 4 * c) = p;
          } else {  // the repeated floats may be another group's: its own slot writes them
            const int e0 = H - 4;
            for (int j = 4 * c - e0; j < 4; ++j) q[e0 + j] = (uint8_t)(p >> (8 * j));
          }
        } else {
          st_stream<NTS>(p, reinterpret_cast<uint32_t*>(q) + c);
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// VJP, a row in the registers of TPR threads, blocks walking the rows with the
// next row's three operands in flight; a block's column partials of dw go to
// part (a block a CU, so that there are 256 partial rows to add up, 4.7 us), or for
// few rows to blocks of their own (few_columns). HBM bounds it: (16384, 4096) 171 us,
// 6.2 TB/s; (8192, 1003) 25 us, 5.4 TB/s; (4096, 16384), on 1024 threads with 8 to 20
// bytes a lane spilled in the exact derivative, 191-193 us in all, 5.6 TB/s.

template <int TPR, int NV>
constexpr int add_bwd_threads() { return TPR == 64 ? (NV <= 2 ? 1024 : 512) : TPR; }

// dx may be gh: every float of it is written by the thread that read it there.
template <int TPR, int NV, int MODE, int KIND, bool NTS, bool FEW>
__global__ __launch_bounds__((add_bwd_threads<TPR, NV>())) void add_norm_bwd_k(
    const float* __restrict__ h, const float* __restrict__ w, const float* __restrict__ rstd,
    const float* __restrict__ gy, const float* gh, float* dx, float* __restrict__ part, int64_t rows, int H_arg,
    float* __restrict__ dw, int row_blocks) {
  const int H = KIND == ROW_FULL ? 4 * TPR * NV : H_arg;
  constexpr bool ODD = KIND == ROW_ODD;
  constexpr int NT = add_bwd_threads<TPR, NV>();
  constexpr int GPB = NT / TPR;
  constexpr int ROWF = TPR * NV * 4;
  if constexpr (FEW) {
    if ((int)blockIdx.x >= row_blocks) {
      few_columns<GPB, false, ACT_NONE>((int)blockIdx.x - row_blocks, h, w, nullptr, nullptr, rstd, gy, dw, nullptr,
                                        (int)rows, H, NT / 64);
      return;
    }
  }
  __shared__ float lds[2 * (NT / 64)];
  __shared__ float comb[GPB > 1 && !FEW ? GPB * ROWF : 1];
  const int t = threadIdx.x % TPR;
  const int gi = threadIdx.x / TPR;
  const int h4 = row_slots<KIND>(H);
  const float inv_n = 1.0f / (float)H;
  const f4* w4 = reinterpret_cast<const f4*>(w);
  const f4 zero = {0.f, 0.f, 0.f, 0.f};
  f4 pdw[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) pdw[k] = zero;
  // the weights stay out of the row loop: in registers, or in LDS where many
  // waves share them or no registers are left (rows of 1024 threads)
  constexpr bool REG_W = TPR > 64 && TPR < 1024;
  constexpr int WL = REG_W ? 1 : TPR * NV;
  __shared__ f4 wl[WL];
  f4 wr[NV];
  auto w_of = [&](int c) -> f4 {
    const int cc = min(c, h4 - 1);
    return c >= h4 ? zero : !w ? f4{1.f, 1.f, 1.f, 1.f} : ODD ? ld_odd(w, H, cc) : w4[cc];
  };
  if constexpr (REG_W) {
#pragma unroll
    for (int k = 0; k < NV; ++k) wr[k] = w_of(k * TPR + t);
  } else {
    for (int c = threadIdx.x; c < WL; c += NT) wl[c] = w_of(c);
    __syncthreads();
  }
  auto w_at = [&](int k) -> f4 {
    if constexpr (REG_W) return wr[k];
    else return wl[k * TPR + t];
  };
  const int64_t ngroups = (int64_t)(FEW ? row_blocks : gridDim.x) * GPB;
  int64_t row = (int64_t)blockIdx.x * GPB + gi;
  int red = 0;
  auto slot = [&]() { return lds + ((red++ & 1) ? NT / 64 : 0); };
  struct Rows {
    RowTile<TPR, NV> x, g, a;
    float inv;
  };
  auto fetch = [&](Rows& f, int64_t q) {
    q = q < rows ? q : rows - 1;
    if constexpr (ODD) {
      f.x.load_odd_clamped(h + q * H, H, t);
      f.g.load_odd_clamped(gy + q * H, H, t);
      f.a.load_odd_clamped(gh + q * H, H, t);
    } else {
      f.x.load_clamped(h + q * H, h4, t);
      f.g.load_clamped(gy + q * H, h4, t);
      f.a.load_clamped(gh + q * H, h4, t);
    }
    f.inv = rstd[q];
  };
  auto process = [&](Rows& f, int64_t q) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = k * TPR + t;
      f4 xh = f.x.v[k] * f.inv;
      f4 g = f.g.v[k];
      if (c >= h4) {
        xh = zero;
        g = zero;
      }
      f.x.v[k] = xh;
      pdw[k] = pdw[k] + without_dup<KIND>(g, H, c) * xh;
      g = g * w_at(k);
      f.g.v[k] = g;
      if constexpr (MODE == OXI_NORM_VJP_EXACT) s += sum4(without_dup<KIND>(g, H, c) * xh);
    }
    if (!dx) return;
    if constexpr (MODE == OXI_NORM_VJP_EXACT) {
      const float a = rsum1<TPR>(s, slot()) * inv_n;
#pragma unroll
      for (int k = 0; k < NV; ++k) f.g.v[k] = f.a.v[k] + (f.g.v[k] - f.x.v[k] * a) * f.inv;
    } else {
#pragma unroll
      for (int k = 0; k < NV; ++k) f.g.v[k] = f.a.v[k] + f.g.v[k] * f.inv;
    }
    if constexpr (ODD) store_owned(f.g, dx + q * H, H, h4, t);
    else f.g.template store<NTS>(dx + q * H, h4, t);
  };
  Rows a, b;
  if constexpr (FEW || TPR == 1024) {  // one row a group, or no registers for a second
#pragma unroll 1
    for (; row < rows; row += ngroups) {
      fetch(a, row);
      process(a, row);
    }
    if constexpr (FEW) return;
  } else {
    fetch(a, row);
    while (row < rows) {
      fetch(b, row + ngroups);
      __builtin_amdgcn_sched_barrier(0);  // the current row's first use stays below the next row's loads
      process(a, row);
      row += ngroups;
      if (row >= rows) break;
      fetch(a, row + ngroups);
      __builtin_amdgcn_sched_barrier(0);
      process(b, row);
      row += ngroups;
    }
  }
  if (!part) return;
  float* pw = part + (int64_t)blockIdx.x * H;
  if constexpr (GPB == 1) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = k * TPR + t;
      if (c >= h4) continue;
      if constexpr (ODD) {
        const int e0 = min(4 * c, H - 4);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (e0 + j >= 4 * c) pw[e0 + j] = pdw[k][j];
      } else {
        reinterpret_cast<f4*>(pw)[c] = pdw[k];
      }
    }
  } else {  // the block's groups in order
#pragma unroll
    for (int k = 0; k < NV; ++k) reinterpret_cast<f4*>(comb + gi * ROWF)[k * TPR + t] = pdw[k];
    __syncthreads();
    for (int c = threadIdx.x; c < H; c += NT) {
      const int e = ODD && c >= (H & ~3) ? 4 * h4 - H + c : c;  // an odd row's last floats end its last slot
      float sum = comb[e];
#pragma unroll
      for (int q = 1; q < GPB; ++q) sum += comb[q * ROWF + e];
      pw[c] = sum;
    }
  }
}

// ---------------------------------------------------------------------------
// Rows that the register kernels do not take (fewer than 4 floats, or more than
// they hold): a block a row, which it walks twice, the second time from the caches.

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

// Four columns a thread, one where the row's are not whole 4-byte words: (8192, 4096)
// in groups of 128 27 us, 6.3 TB/s; (8192, 1003) 19 us, a byte a thread.
template <int W>
__global__ __launch_bounds__(BS) void e4m3_dequantize_k(const uint8_t* __restrict__ q, const float* __restrict__ scale,
                                                        float* __restrict__ y, int64_t rows, int H, int group,
                                                        int groups) {
  const int c = (blockIdx.x * BS + threadIdx.x) * W;
  if (c >= H) return;
  const int g = c / group;  // groups are multiples of 4 columns, or the row
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float s = scale[row * groups + g];
    if constexpr (W == 4) {
      const int p = *reinterpret_cast<const int*>(q + row * H + c);
      const f4 v = {__builtin_amdgcn_cvt_f32_fp8(p, 0), __builtin_amdgcn_cvt_f32_fp8(p, 1),
                    __builtin_amdgcn_cvt_f32_fp8(p, 2), __builtin_amdgcn_cvt_f32_fp8(p, 3)};
      *reinterpret_cast<f4u*>(y + row * H + c) = v * s;
    } else {
      y[row * H + c] = __builtin_amdgcn_cvt_f32_fp8(q[row * H + c], 0) * s;
    }
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

int log_lanes_of(int64_t group, int64_t groups) {
  return groups == 1 ? 0 : group == 32 ? 3 : group == 64 ? 4 : group == 128 ? 5 : 6;
}

template <int OUT, bool NTS>
bool launch_fwd(int cfg, bool odd, const float* x, const float* r, const float* w, float* h, void* out, float* stat,
                int64_t rows, int H, float eps, int log_lanes, int groups) {
  hipStream_t s = stream();
#define OXI_AF_GO(TPR, NV, KIND, NTS_, NT)                                                                      \
  add_norm_fwd_k<TPR, NV, KIND, NTS_, NT, OUT><<<dim3((unsigned)ceil_div(rows, NT / TPR)), dim3(NT), 0, s>>>(   \
      x, r, w, h, out, stat, rows, H, eps, log_lanes, groups)
#define OXI_AF(TPR, NV)                                                                                         \
  case TPR * 10 + NV:                                                                                           \
    if (!grid_fits(ceil_div(rows, row_block_threads(TPR) / TPR), row_block_threads(TPR))) return false;         \
    if (odd) OXI_AF_GO(TPR, NV, ROW_ODD, false, row_block_threads(TPR));                                        \
    else if (H == 4 * TPR * NV) OXI_AF_GO(TPR, NV, ROW_FULL, NTS, row_block_threads(TPR));                      \
    else OXI_AF_GO(TPR, NV, ROW_VEC, NTS, row_block_threads(TPR));                                              \
    return true;
  switch (cfg) {
    OXI_AF(64, 1)
    OXI_AF(64, 2)
    OXI_AF(64, 3)
    OXI_AF(64, 4)
    OXI_AF(256, 2)
    OXI_AF(256, 4)
    OXI_AF(256, 8)
    OXI_AF(1024, 4)
  }
#undef OXI_AF
#undef OXI_AF_GO
  return false;
}

// The VJP's launch: its row configuration (0: the loop kernel), threads and
// blocks, and whether dw is formed in the same launch.
struct BwdShape {
  int cfg, nt;
  int64_t nblk;
  bool few;
};
BwdShape bwd_shape(int64_t rows, int64_t H) {
  BwdShape b;
  b.cfg = plain_bwd_cfg(H);
  const int tpr = b.cfg ? b.cfg / 10 : BS;
  b.nt = tpr == 64 ? (b.cfg % 10 <= 2 ? 1024 : 512) : tpr;  // add_bwd_threads
  b.nblk = std::min<int64_t>(ceil_div(rows, b.nt / tpr), cu_count());
  b.few = b.cfg && rows <= FEW_MAX && rows <= b.nblk * (b.nt / tpr);
  return b;
}

template <int MODE, bool NTS>
void launch_bwd_cfg(const BwdShape& b, bool odd, const float* h, const float* w, const float* rstd, const float* gy,
                    const float* gh, float* dx, float* part, int64_t rows, int H, float* dw) {
  hipStream_t s = stream();
#define OXI_AB_GO(TPR, NV, KIND, NTS_, FEW, BLOCKS)                                                            \
  add_norm_bwd_k<TPR, NV, MODE, KIND, NTS_, FEW><<<dim3((unsigned)(BLOCKS)), dim3(b.nt), 0, s>>>(              \
      h, w, rstd, gy, gh, dx, part, rows, H, dw, (int)b.nblk)
#define OXI_AB(TPR, NV)                                                                                        \
  case TPR * 10 + NV:                                                                                          \
    if (b.few && dw) {                                                                                         \
      if (odd) OXI_AB_GO(TPR, NV, ROW_ODD, false, true, b.nblk + ceil_div(H, 64));                             \
      else OXI_AB_GO(TPR, NV, ROW_VEC, false, true, b.nblk + ceil_div(H, 64));                                 \
    } else if (odd) {                                                                                          \
      OXI_AB_GO(TPR, NV, ROW_ODD, false, false, b.nblk);                                                       \
    } else if (H == 4 * TPR * NV) {                                                                            \
      OXI_AB_GO(TPR, NV, ROW_FULL, NTS, false, b.nblk);                                                        \
    } else {                                                                                                   \
      OXI_AB_GO(TPR, NV, ROW_VEC, NTS, false, b.nblk);                                                         \
    }                                                                                                          \
    return;
  switch (b.cfg) {
    OXI_AB(64, 1)
    OXI_AB(64, 2)
    OXI_AB(64, 3)
    OXI_AB(64, 4)
    OXI_AB(256, 2)
    OXI_AB(512, 2)
    OXI_AB(512, 4)
    OXI_AB(1024, 4)
  }
#undef OXI_AB
#undef OXI_AB_GO
  add_norm_bwd_loop_k<MODE><<<dim3((unsigned)b.nblk), dim3(BS), 0, s>>>(h, w, rstd, gy, gh, dx, part, rows, H);
}

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
  const int cfg = norm_fwd_cfg(rows, cols);
  const bool odd = !vec_ok(cols, {x, r, w, h, y});
  const bool done = nt_stream_stores(rows * cols * 8)
                        ? launch_fwd<OUT_F32, true>(cfg, odd, x, r, w, h, y, rstd, rows, (int)cols, eps, 0, 0)
                        : launch_fwd<OUT_F32, false>(cfg, odd, x, r, w, h, y, rstd, rows, (int)cols, eps, 0, 0);
  if (!done)
    add_norm_fwd_loop_k<<<dim3((unsigned)walk_blocks(rows)), dim3(BS), 0, stream()>>>(x, r, w, h, y, rstd, rows,
                                                                                     (int)cols, eps);
  return check_launch("add_rms_norm_fwd");
}

int oxi_add_rms_norm_bwd_workspace(int64_t rows, int64_t cols, int64_t* bytes) {
  if (int rc = check_sizes("add_rms_norm_bwd_workspace", rows, cols)) return rc;
  if (!bytes) return fail(OXI_INVALID_ARGUMENT, "add_rms_norm_bwd_workspace: NULL result pointer");
  OXI_CHECK_INIT();
  // the norm's own VJP, for a call without gh, keeps two planes of partials
  const int64_t own = rows && cols ? (int64_t)sizeof(float) * bwd_shape(rows, cols).nblk * cols : 0;
  const int64_t plain = rows && cols ? (int64_t)bwd_part_bytes(true, rows, cols, plain_bwd_cfg(cols)) : 0;
  *bytes = std::max(own, plain);
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
    if (reinterpret_cast<uintptr_t>(workspace) & 15u)
      return fail(OXI_INVALID_ARGUMENT, "add_rms_norm_bwd: the workspace at %p is not 16-byte aligned", workspace);
  }
  OXI_CHECK_INIT();
  if (rows == 0 || cols == 0) return dw && cols ? oxi_fill(dw, cols, 0.f) : OXI_OK;
  if (!dx && !dw) return OXI_OK;
  if (!gh) {
    const size_t fixed = workspace ? bwd_part_bytes(true, rows, cols, plain_bwd_cfg(cols)) : 0;
    return norm_bwd_none(false, mode, NormBwdArgs{h, w, nullptr, nullptr, rstd, gy, nullptr, dx, dw, nullptr, rows,
                                                  cols, workspace, nullptr, 0, fixed});
  }
  const BwdShape b = bwd_shape(rows, cols);
  const bool parts = dw && !b.few;
  Workspace ws(parts && !workspace ? sizeof(float) * (size_t)b.nblk * (size_t)cols : 0);
  float* part = !parts ? nullptr : workspace ? static_cast<float*>(workspace) : ws.as<float>();
  if (parts && !part) return fail_alloc("add_rms_norm_bwd: column partials");
  const bool odd = !vec_ok(cols, {h, w, gy, gh, dx});
  const int H = (int)cols;
  const bool nt = nt_stream_stores(rows * cols * 4);
#define OXI_AB_MODE(MODE)                                                                         \
  if (nt) launch_bwd_cfg<MODE, true>(b, odd, h, w, rstd, gy, gh, dx, part, rows, H, dw);          \
  else launch_bwd_cfg<MODE, false>(b, odd, h, w, rstd, gy, gh, dx, part, rows, H, dw);
  if (mode == OXI_NORM_VJP_REF) {
    OXI_AB_MODE(OXI_NORM_VJP_REF)
  } else {
    OXI_AB_MODE(OXI_NORM_VJP_EXACT)
  }
#undef OXI_AB_MODE
  if (int rc = check_launch("add_rms_norm_bwd")) return rc;
  if (!parts) return OXI_OK;
  const dim3 fg((unsigned)ceil_div(cols, FIN_C), 1);
  col_finish_k<16><<<fg, dim3(FIN_C * 16), 0, stream()>>>(part, (int)b.nblk, H, dw, nullptr);
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
  const int64_t groups = ceil_div(cols, group);
  const int cfg = norm_fwd_cfg(rows, cols);
  const bool odd = !vec_ok(cols, {x, r, w, r ? h : nullptr}) || (reinterpret_cast<uintptr_t>(q) & 3u);
  const int lanes = log_lanes_of(group, groups);
  const bool done =
      nt_stream_stores(rows * cols * (r ? 5 : 1))
          ? launch_fwd<OUT_E4M3, true>(cfg, odd, x, r, w, h, q, scale, rows, (int)cols, eps, lanes, (int)groups)
          : launch_fwd<OUT_E4M3, false>(cfg, odd, x, r, w, h, q, scale, rows, (int)cols, eps, lanes, (int)groups);
  if (done) return check_launch("add_rms_norm_e4m3_fwd");
  add_norm_e4m3_loop_k<<<dim3((unsigned)walk_blocks(rows)), dim3(BS), 0, stream()>>>(
      x, r, w, h, q, scale, rows, (int)cols, (int)group, (int)groups, eps);
  return check_launch("add_rms_norm_e4m3_fwd");
}

int oxi_e4m3_dequantize(const uint8_t* q, const float* scale, float* y, int64_t rows, int64_t cols, int64_t group) {
  if (int rc = check_sizes("e4m3_dequantize", rows, cols)) return rc;
  if (rows == 0 || cols == 0) return OXI_OK;
  if (int rc = check_group("e4m3_dequantize", cols, group)) return rc;
  if (!q || !scale || !y) return fail(OXI_INVALID_ARGUMENT, "e4m3_dequantize: NULL tensor pointer");
  OXI_CHECK_INIT();
  const int groups = (int)ceil_div(cols, group);
  const unsigned gy = (unsigned)std::min<int64_t>(rows, 16384);
  if (cols % 4 == 0 && !(reinterpret_cast<uintptr_t>(q) & 3u))
    e4m3_dequantize_k<4><<<dim3((unsigned)ceil_div(cols, 4 * BS), gy), dim3(BS), 0, stream()>>>(
        q, scale, y, rows, (int)cols, (int)group, groups);
  else
    e4m3_dequantize_k<1><<<dim3((unsigned)ceil_div(cols, BS), gy), dim3(BS), 0, stream()>>>(
        q, scale, y, rows, (int)cols, (int)group, groups);
  return check_launch("e4m3_dequantize");
}

}  // extern "C"

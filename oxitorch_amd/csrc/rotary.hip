// Rotary positions for gfx950: pairs (u, v) of the first `rot` elements of each
// head turn by an angle a = position * inv_freq[i], the others are copied.
//
//   (u, v) -> scale * (u cos a - v sin a, v cos a + u sin a)
//
// The angle is formed and reduced in 64 bits: at position 10^6 a 32-bit product
// is off by up to 0.06. A token's heads share its angles.
#include "internal.h"

namespace oxi {
namespace {

constexpr int BS = 256;

struct RotaryArgs {
  const float* x;
  float* y;
  int64_t xs[4], ys[4];  // strides of (batch, token, head, element)
  int64_t tokens, heads;
  int64_t ps[2];  // strides of the positions
  const int64_t* positions;
  int64_t offset;
  const double* inv_freq;
  int dim, half;  // elements a head, pairs that turn
  int interleaved;
  float sign, scale;
};

__device__ __forceinline__ int64_t position_of(const RotaryArgs& a, int64_t b, int64_t t) {
  return a.offset + (a.positions ? a.positions[b * a.ps[0] + t * a.ps[1]] : t);
}

// A thread a pair (or copied element) of a token, all heads.
__global__ __launch_bounds__(BS) void rotary_k(const RotaryArgs a, int64_t n, int units) {
  const int64_t step = (int64_t)gridDim.x * BS;
  for (int64_t i = (int64_t)blockIdx.x * BS + threadIdx.x; i < n; i += step) {
    const int j = (int)(i % units);
    const int64_t bt = i / units;
    const int64_t b = bt / a.tokens, t = bt % a.tokens;
    const float* x = a.x + b * a.xs[0] + t * a.xs[1];
    float* y = a.y + b * a.ys[0] + t * a.ys[1];
    if (j < a.half) {
      double sn, cs;
      sincos((double)position_of(a, b, t) * a.inv_freq[j], &sn, &cs);
      const float c = (float)(cs * (double)a.scale), s = (float)(sn * (double)a.scale) * a.sign;
      const int e0 = a.interleaved ? 2 * j : j, e1 = a.interleaved ? 2 * j + 1 : j + a.half;
      for (int64_t k = 0; k < a.heads; ++k) {
        const float u = x[k * a.xs[2] + e0 * a.xs[3]], v = x[k * a.xs[2] + e1 * a.xs[3]];
        y[k * a.ys[2] + e0 * a.ys[3]] = u * c - v * s;
        y[k * a.ys[2] + e1 * a.ys[3]] = v * c + u * s;
      }
    } else {
      const int64_t e = a.half + j;  // rot + (j - half)
      for (int64_t k = 0; k < a.heads; ++k) y[k * a.ys[2] + e * a.ys[3]] = x[k * a.xs[2] + e * a.xs[3]];
    }
  }
}

}  // namespace
}  // namespace oxi

using namespace oxi;

extern "C" {

int oxi_rotary(const float* x, const int64_t* x_strides, float* y, const int64_t* y_strides, const int64_t* shape,
               const int64_t* positions, const int64_t* pos_strides, int64_t offset, const double* inv_freq,
               int64_t rot, int layout, int inverse, float scale) {
  if (!shape || !x_strides || !y_strides) return fail(OXI_INVALID_ARGUMENT, "rotary: NULL shape or strides");
  int64_t n = 1;
  for (int d = 0; d < 4; ++d) {
    if (shape[d] < 0) return fail(OXI_INVALID_ARGUMENT, "rotary: negative size");
    if (shape[d] && n > ((int64_t)1 << 60) / shape[d])
      return fail(OXI_INVALID_ARGUMENT, "rotary: size exceeds the kernel limits");
    n *= shape[d] ? shape[d] : 1;
  }
  const int64_t dim = shape[3];
  if (dim > ((int64_t)1 << 20)) return fail(OXI_INVALID_ARGUMENT, "rotary: heads of %lld elements exceed the kernel "
                                                                   "limits", (long long)dim);
  if (rot < 0 || rot > dim || rot % 2)
    return fail(OXI_INVALID_ARGUMENT, "rotary: %lld elements of a head of %lld to turn: an even number, at most all",
                (long long)rot, (long long)dim);
  if (layout != OXI_ROTARY_HALF && layout != OXI_ROTARY_INTERLEAVED)
    return fail(OXI_INVALID_ARGUMENT, "rotary: unknown layout %d", layout);
  if (positions && !pos_strides) return fail(OXI_INVALID_ARGUMENT, "rotary: positions without strides");
  for (int d = 0; d < 4; ++d)
    if (shape[d] == 0) return OXI_OK;
  if (!x || !y || (rot && !inv_freq)) return fail(OXI_INVALID_ARGUMENT, "rotary: NULL tensor pointer");
  for (int d = 0; d < 4; ++d) {
    if (shape[d] > 1 && y_strides[d] == 0) return fail(OXI_INVALID_ARGUMENT, "rotary: y is a broadcast view");
    if (x == y && shape[d] > 1 && x_strides[d] != y_strides[d])
      return fail(OXI_INVALID_ARGUMENT, "rotary: in place, y has to have x's strides");
  }
  OXI_CHECK_INIT();
  RotaryArgs a;
  a.x = x;
  a.y = y;
  for (int d = 0; d < 4; ++d) {
    a.xs[d] = x_strides[d];
    a.ys[d] = y_strides[d];
  }
  a.tokens = shape[1];
  a.heads = shape[2];
  a.ps[0] = positions ? pos_strides[0] : 0;
  a.ps[1] = positions ? pos_strides[1] : 0;
  a.positions = positions;
  a.offset = offset;
  a.inv_freq = inv_freq;
  a.dim = (int)dim;
  a.half = (int)(rot / 2);
  a.interleaved = layout == OXI_ROTARY_INTERLEAVED;
  a.sign = inverse ? -1.f : 1.f;
  a.scale = scale;
  const int units = (int)(dim - rot / 2);
  const int64_t work = shape[0] * shape[1] * units;
  const int64_t blocks = ceil_div(work, BS) < 65536 ? ceil_div(work, BS) : 65536;
  rotary_k<<<dim3((unsigned)blocks), dim3(BS), 0, stream()>>>(a, work, units);
  return check_launch("rotary");
}

}  // extern "C"

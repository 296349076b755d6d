// Rotary positions for gfx950: pairs (u, v) of the first `rot` elements of each
// head turn by an angle a = position * inv_freq[i], the others are copied.
//
//   (u, v) -> scale * (u cos a - v sin a, v cos a + u sin a)
//
// The angle is formed and reduced in 64 bits: at position 10^6 a 32-bit product
// is off by up to 0.06. A block takes a few tokens with some or all of their
// heads: its threads first form the tokens' cosines and sines, once for all
// heads, in LDS, then stream the heads through registers in units of 2W
// elements (W pairs, or 2W elements that are copied), four units in flight.
#include <algorithm>

#include "internal.h"
#include "rowtile.h"

namespace oxi {
namespace {

constexpr int BS = 256;
constexpr int MAX_DIM = 8192;    // elements a head
constexpr int MAX_TOKENS = 64;   // tokens a block
constexpr int ANGLES = 2048;     // cosines a block forms, when one token's fit

// n / d for n * d < 2^32: the high half of n * ceil(2^32 / d).
struct Divider {
  uint32_t d, m;
};
Divider divider(uint32_t d) { return {d, d > 1 ? (uint32_t)((((uint64_t)1 << 32) + d - 1) / d) : 0}; }
__device__ __forceinline__ uint32_t quotient(uint32_t n, const Divider& v) { return v.d > 1 ? __umulhi(n, v.m) : n; }

struct RotaryArgs {
  const float* x;
  float* y;
  int64_t xs[4], ys[4];  // strides of (batch, token, head, element)
  int64_t tokens, all;   // tokens a sequence, and of all of them
  int64_t ps[2];         // strides of the positions
  const int64_t* positions;
  int64_t offset;
  const double* inv_freq;
  int heads, dim, half;  // heads; elements a head; pairs that turn
  int interleaved;
  float scale, sin_scale;
  int block_tokens, block_heads;
  int token_first;         // units go through a head's tokens before its next head
  Divider units, inner;    // units a head; tokens or heads, whichever go first
};

// cos and sin of 2 pi r, |r| <= 1/2: the nearest quarter turn taken off, both
// series on what is left (at most pi/4: the terms left out are below 2^-28).
__device__ __forceinline__ void cos_sin_turn(double r, float& c, float& s) {
  const double q = rint(r * 4.0);
  const float x = (float)((r - q * 0.25) * 6.283185307179586);
  const float z = x * x;
  float ps = fmaf(z, 1.f / 362880.f, -1.f / 5040.f);
  ps = fmaf(ps, z, 1.f / 120.f);
  ps = fmaf(ps, z, -1.f / 6.f);
  const float sx = fmaf(ps * z, x, x);
  float pc = fmaf(z, -1.f / 3628800.f, 1.f / 40320.f);
  pc = fmaf(pc, z, -1.f / 720.f);
  pc = fmaf(pc, z, 1.f / 24.f);
  pc = fmaf(pc, z, -0.5f);
  const float cx = fmaf(pc, z, 1.f);
  const int k = (int)q & 3;
  const float a = k & 1 ? sx : cx, b = k & 1 ? cx : sx;
  c = k == 1 || k == 2 ? -a : a;
  s = k >= 2 ? -b : b;
}

template <int W>
struct Vec {
  typedef float T __attribute__((ext_vector_type(W), aligned(4)));
};
template <>
struct Vec<1> {
  typedef float T;
};

template <int W, bool NTS>
__device__ __forceinline__ void put(typename Vec<W>::T v, float* p) {
  typedef typename Vec<W>::T V;
  if constexpr (NTS) __builtin_nontemporal_store(v, reinterpret_cast<V*>(p));
  else *reinterpret_cast<V*>(p) = v;
}

// W: pairs a unit. STRIDED: elements lie apart (W = 1 only).
template <int W, bool STRIDED, bool NTS>
__global__ __launch_bounds__(BS) void rotary_k(const RotaryArgs g) {
  typedef typename Vec<W>::T V;
  constexpr int U = 4;  // units in flight a thread
  extern __shared__ __align__(16) float lds[];  // block_tokens x half cosines, then as many sines
  __shared__ int64_t xbase[MAX_TOKENS], ybase[MAX_TOKENS];
  const int64_t i0 = (int64_t)blockIdx.x * g.block_tokens;
  const int nt = (int)min((int64_t)g.block_tokens, g.all - i0);
  const int head0 = blockIdx.y * g.block_heads;
  const int nh = min(g.block_heads, g.heads - head0);
  float* const cs = lds;
  float* const sn = lds + g.block_tokens * g.half;
  for (int j = threadIdx.x; j < nt; j += BS) {
    const int64_t b = (i0 + j) / g.tokens, t = (i0 + j) % g.tokens;
    xbase[j] = b * g.xs[0] + t * g.xs[1] + head0 * g.xs[2];
    ybase[j] = b * g.ys[0] + t * g.ys[1] + head0 * g.ys[2];
  }
  for (int j = threadIdx.x; j < nt * g.half; j += BS) {
    const int k = j / g.half, i = j - k * g.half;
    const int64_t b = (i0 + k) / g.tokens, t = (i0 + k) % g.tokens;
    const int64_t pos = g.offset + (g.positions ? g.positions[b * g.ps[0] + t * g.ps[1]] : t);
    const double a = (double)pos * g.inv_freq[i] * 0.15915494309189535;  // turns
    float c, s;
    cos_sin_turn(a - rint(a), c, s);
    cs[j] = c * g.scale;
    sn[j] = s * g.sin_scale;
  }
  __syncthreads();
  const uint32_t nu = g.units.d;
  const uint32_t turning = g.half / W;
  // a last block's tokens, or heads, may be fewer than the divider's
  for (uint32_t n0 = threadIdx.x; n0 < (uint32_t)g.block_tokens * g.block_heads * nu; n0 += U * BS) {
    V a[U], b[U];
    const float* xp[U];
    float* yp[U];
    int tok[U];
    int e0[U], e1[U];
    uint32_t unit[U];
    bool in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t q = n0 + u * BS;
      const uint32_t r = quotient(q, g.units);
      unit[u] = q - r * nu;
      const uint32_t o = quotient(r, g.inner), i = r - o * g.inner.d;
      tok[u] = g.token_first ? i : o;
      const int head = g.token_first ? o : i;
      in[u] = tok[u] < nt && head < nh;
      const bool turn = unit[u] < turning;
      const int p = unit[u] * W;  // first pair, or half the first element of a copied unit
      e0[u] = turn && !g.interleaved ? p : 2 * p;
      e1[u] = turn && !g.interleaved ? p + g.half : 2 * p + W;
      if (!in[u]) continue;
      xp[u] = g.x + xbase[tok[u]] + head * g.xs[2];
      yp[u] = g.y + ybase[tok[u]] + head * g.ys[2];
      if constexpr (STRIDED) {
        a[u] = xp[u][e0[u] * g.xs[3]];
        if (e1[u] < g.dim) b[u] = xp[u][e1[u] * g.xs[3]];
      } else {
        a[u] = *reinterpret_cast<const V*>(xp[u] + e0[u]);
        if (W > 1 || e1[u] < g.dim) b[u] = *reinterpret_cast<const V*>(xp[u] + e1[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!in[u]) continue;
      if (unit[u] < turning) {
        const float* c = cs + tok[u] * g.half + unit[u] * W;
        const float* s = sn + tok[u] * g.half + unit[u] * W;
        if constexpr (W == 1) {
          const float p = a[u], q = b[u];
          a[u] = p * c[0] - q * s[0];
          b[u] = q * c[0] + p * s[0];
        } else if (g.interleaved) {
#pragma unroll
          for (int j = 0; j < W; j += 2) {
            const float p = a[u][j], q = a[u][j + 1];
            a[u][j] = p * c[j / 2] - q * s[j / 2];
            a[u][j + 1] = q * c[j / 2] + p * s[j / 2];
            const float p2 = b[u][j], q2 = b[u][j + 1];
            b[u][j] = p2 * c[(W + j) / 2] - q2 * s[(W + j) / 2];
            b[u][j + 1] = q2 * c[(W + j) / 2] + p2 * s[(W + j) / 2];
          }
        } else {
#pragma unroll
          for (int j = 0; j < W; ++j) {
            const float p = a[u][j], q = b[u][j];
            a[u][j] = p * c[j] - q * s[j];
            b[u][j] = q * c[j] + p * s[j];
          }
        }
      }
      if constexpr (STRIDED) {
        yp[u][e0[u] * g.ys[3]] = a[u];
        if (e1[u] < g.dim) yp[u][e1[u] * g.ys[3]] = b[u];
      } else {
        put<W, NTS>(a[u], yp[u] + e0[u]);
        if (W > 1 || e1[u] < g.dim) put<W, NTS>(b[u], yp[u] + e1[u]);
      }
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
  if (dim > MAX_DIM || shape[2] > ((int64_t)1 << 20))
    return fail(OXI_INVALID_ARGUMENT, "rotary: %lld heads of %lld elements exceed the kernel limits",
                (long long)shape[2], (long long)dim);
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
  a.all = shape[0] * shape[1];
  a.ps[0] = positions ? pos_strides[0] : 0;
  a.ps[1] = positions ? pos_strides[1] : 0;
  a.positions = positions;
  a.offset = offset;
  a.inv_freq = inv_freq;
  a.heads = (int)shape[2];
  a.dim = (int)dim;
  a.half = (int)(rot / 2);
  a.interleaved = layout == OXI_ROTARY_INTERLEAVED;
  a.scale = scale;
  a.sin_scale = inverse ? -scale : scale;
  const bool strided = (dim > 1 && (x_strides[3] != 1 || y_strides[3] != 1));
  int w = strided ? 1 : 4;
  while (w > 1 && (a.half % w || (dim - rot) % (2 * w))) w /= 2;
  const int64_t units = ceil_div(dim - rot, 2 * w) + a.half / w;
  // A block's work: tokens and heads of about 8 units a thread where there are
  // enough blocks for every CU at that, down to one unit a thread.
  int64_t goal = 8 * BS;
  while (goal > BS && a.all * a.heads * units < goal * 2 * cu_count()) goal /= 2;
  int64_t heads = std::min<int64_t>(a.heads, std::max<int64_t>(1, goal / units));
  int64_t tokens = std::max<int64_t>(1, goal / (heads * units));
  tokens = std::min<int64_t>(std::min<int64_t>(tokens, MAX_TOKENS), a.half ? std::max(1, ANGLES / a.half) : MAX_TOKENS);
  tokens = std::min<int64_t>(tokens, a.all);
  a.block_tokens = (int)tokens;
  a.block_heads = (int)heads;
  a.token_first = shape[1] > 1 && x_strides[1] < x_strides[2];
  a.units = divider((uint32_t)units);
  a.inner = divider((uint32_t)(a.token_first ? tokens : heads));
  const int64_t bx = ceil_div(a.all, tokens), by = ceil_div(a.heads, heads);
  if (!grid_fits(bx, BS) || by > 65535)
    return fail(OXI_INVALID_ARGUMENT, "rotary: size exceeds the kernel limits");
  const dim3 grid((unsigned)bx, (unsigned)by);
  const size_t lds = sizeof(float) * 2 * (size_t)tokens * (size_t)a.half;
  const bool nts = nt_stores(n * 4);
#define OXI_ROT(W, STRIDED)                                                          \
  if (nts) rotary_k<W, STRIDED, true><<<grid, dim3(BS), lds, stream()>>>(a);         \
  else rotary_k<W, STRIDED, false><<<grid, dim3(BS), lds, stream()>>>(a);
  if (strided) {
    OXI_ROT(1, true)
  } else if (w == 4) {
    OXI_ROT(4, false)
  } else if (w == 2) {
    OXI_ROT(2, false)
  } else {
    OXI_ROT(1, false)
  }
#undef OXI_ROT
  return check_launch("rotary");
}

}  // extern "C"

// Rotary positions for gfx950: pairs (u, v) of the first `rot` elements of each
// head turn by an angle a = position * inv_freq[i], the others are copied.
//
//   (u, v) -> scale * (u cos a - v sin a, v cos a + u sin a)
//
// The angle is formed and reduced in 64 bits: at position 10^6 a 32-bit product
// is off by up to 0.06. A block takes a few tokens with some or all of their
// heads. A head is cut into units of 2W elements (W pairs, or 2W elements that
// are copied); a thread has one unit, of some of the block's (token, head) rows,
// ROWS of them in flight. The first of them are loaded before the block forms its
// tokens' cosines and sines, once for all heads, in LDS. HBM bounds it: (4, 4096,
// 32, 128) 87 us a call, 6.1 TB/s; (16, 1023, 12, 64) heads first 22 us, 4.6 TB/s,
// where a launch's beginning and end weigh.
#include <algorithm>

#include "internal.h"
#include "launch_limits.h"
#include "rowtile.h"

namespace oxi {
namespace {

constexpr int BS = 256;
constexpr int MAX_DIM = 8192;    // elements a head
constexpr int MAX_TOKENS = 64;   // tokens a block
constexpr int ANGLES = 2048;     // cosines a block forms, when one token's fit
constexpr int ROWS = 2;

struct RotaryArgs {
  const float* x;
  float* y;
  int64_t xs[4], ys[4];  // strides of (batch, token, head, element)
  uint32_t tokens, all;  // tokens a sequence, and of all of them
  int64_t ps[2];         // strides of the positions
  const int64_t* positions;
  int64_t offset;
  const double* inv_freq;
  int heads, dim, half;  // heads; elements a head; pairs that turn
  int interleaved;
  float scale, sin_scale;
  int block_tokens, block_heads;
  int units;        // units a head
  int token_first;  // a thread's rows go through a head's tokens before its next head
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
  typedef float Whole __attribute__((ext_vector_type(W)));  // at its own alignment: LDS
};
template <>
struct Vec<1> {
  typedef float T, Whole;
};

template <int W, bool NTS>
__device__ __forceinline__ void put(typename Vec<W>::T v, float* p) {
  typedef typename Vec<W>::T V;
  if constexpr (NTS) __builtin_nontemporal_store(v, reinterpret_cast<V*>(p));
  else *reinterpret_cast<V*>(p) = v;
}

template <int W>
__device__ __forceinline__ typename Vec<W>::T get(const float* p) {
  typedef typename Vec<W>::T V;
  return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
}

// The W/2 neighbouring pairs of x turned.
template <int W, class H>
__device__ __forceinline__ typename Vec<W>::T turned(typename Vec<W>::T x, H c, H s) {
  if constexpr (W == 2) {
    return {x.x * c - x.y * s, x.y * c + x.x * s};
  } else if constexpr (W == 4) {
    return {x.x * c.x - x.y * s.x, x.y * c.x + x.x * s.x, x.z * c.y - x.w * s.y, x.w * c.y + x.z * s.y};
  } else {
    return x;
  }
}

// W: pairs a unit. STRIDED: elements lie apart (W = 1 only).
template <int W, bool STRIDED, bool NTS>
__global__ __launch_bounds__(BS) void rotary_k(const RotaryArgs g) {
  typedef typename Vec<W>::T V;
  extern __shared__ __align__(16) float lds[];  // block_tokens x half cosines, then as many sines
  __shared__ int64_t xbase[MAX_TOKENS], ybase[MAX_TOKENS];
  const uint32_t i0 = blockIdx.x * (uint32_t)g.block_tokens;
  const int nt = min(g.block_tokens, (int)(g.all - i0));
  const int head0 = blockIdx.y * g.block_heads;
  const int nh = min(g.block_heads, g.heads - head0);
  const int unit0 = blockIdx.z * BS;
  const int nu = min(g.units - unit0, BS);
  float* const cs = lds;
  float* const sn = lds + g.block_tokens * g.half;
  auto position = [&](int k) -> int64_t {
    const uint32_t b = (i0 + k) / g.tokens, t = (i0 + k) % g.tokens;
    return g.offset + (g.positions ? g.positions[b * g.ps[0] + t * g.ps[1]] : (int64_t)t);
  };
  const int angles = nt * g.half;
  int64_t pos = 0;
  double freq = 0.0;
  if ((int)threadIdx.x < angles) {
    pos = position(threadIdx.x / g.half);
    freq = g.inv_freq[threadIdx.x % g.half];
  }
  for (int j = threadIdx.x; j < nt; j += BS) {
    const uint32_t b = (i0 + j) / g.tokens, t = (i0 + j) % g.tokens;
    xbase[j] = b * g.xs[0] + t * g.xs[1] + head0 * g.xs[2];
    ybase[j] = b * g.ys[0] + t * g.ys[1] + head0 * g.ys[2];
  }
  // this thread's unit and the first of its rows; `step` rows on is the next
  const int step = BS / nu;
  const int first = threadIdx.x / nu;
  const int unit = unit0 + threadIdx.x - first * nu;
  const int inner = g.token_first ? nt : nh, outer = g.token_first ? nh : nt;
  const int turning = g.half / W;
  const bool turn = unit < turning;
  // The unit's two vectors: W elements each of the head's turning (or copied)
  // half and of its other half, in the interleaved layout too (W/2 pairs each), so
  // that neighbouring threads read neighbouring vectors; single pairs as they lie.
  const int p = unit * W;
  const int c0 = p - g.half;  // a copied unit's first element past the turning ones
  const int rest = g.dim - 2 * g.half;
  const int e0 = !turn ? 2 * g.half + c0 : W == 1 && g.interleaved ? 2 * p : p;
  const int e1 = !turn ? 2 * g.half + (rest + 1) / 2 + c0 : W == 1 && g.interleaved ? 2 * p + 1 : p + g.half;
  const bool has1 = W > 1 || e1 < g.dim;  // an odd count of copied elements
  int i = first % inner, o = first < step ? first / inner : outer;  // threads past the last whole row: none
  const int di = step % inner, dq = step / inner;
  __syncthreads();
  V a[ROWS], b[ROWS];
  int tok[ROWS], head[ROWS];
  bool in[ROWS];
  auto load = [&]() {
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      in[u] = o < outer;
      tok[u] = g.token_first ? i : o;
      head[u] = g.token_first ? o : i;
      i += di;
      o += dq;
      if (i >= inner) {
        i -= inner;
        ++o;
      }
      if (!in[u]) continue;
      const float* x = g.x + xbase[tok[u]] + head[u] * g.xs[2];
      if constexpr (STRIDED) {
        a[u] = x[e0 * g.xs[3]];
        if (has1) b[u] = x[e1 * g.xs[3]];
      } else {
        a[u] = get<W>(x + e0);
        if (has1) b[u] = get<W>(x + e1);
      }
    }
  };
  load();
  for (int j = threadIdx.x; j < angles; j += BS) {
    if (j != (int)threadIdx.x) {
      pos = position(j / g.half);
      freq = g.inv_freq[j % g.half];
    }
    const double a = (double)pos * freq * 0.15915494309189535;  // turns
    float c, s;
    cos_sin_turn(a - rint(a), c, s);
    cs[j] = c * g.scale;
    sn[j] = s * g.sin_scale;
  }
  __syncthreads();
  while (in[0]) {
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      if (!in[u]) continue;
      if (turn) {
        const float* ct = cs + tok[u] * g.half;
        const float* st = sn + tok[u] * g.half;
        if (W > 1 && g.interleaved) {
          typedef typename Vec<(W > 1 ? W / 2 : 1)>::Whole H;
          const H ca = *reinterpret_cast<const H*>(ct + p / 2), sa = *reinterpret_cast<const H*>(st + p / 2);
          const H cb = *reinterpret_cast<const H*>(ct + (g.half + p) / 2), sb = *reinterpret_cast<const H*>(st + (g.half + p) / 2);
          a[u] = turned<W>(a[u], ca, sa);
          b[u] = turned<W>(b[u], cb, sb);
        } else {
          const V c = *reinterpret_cast<const typename Vec<W>::Whole*>(ct + p);
          const V s = *reinterpret_cast<const typename Vec<W>::Whole*>(st + p);
          const V x = a[u], y = b[u];
          a[u] = x * c - y * s;
          b[u] = y * c + x * s;
        }
      }
      float* y = g.y + ybase[tok[u]] + head[u] * g.ys[2];
      if constexpr (STRIDED) {
        y[e0 * g.ys[3]] = a[u];
        if (has1) y[e1 * g.ys[3]] = b[u];
      } else {
        put<W, NTS>(a[u], y + e0);
        if (has1) put<W, NTS>(b[u], y + e1);
      }
    }
    load();
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
  if (dim > MAX_DIM || shape[2] > ((int64_t)1 << 20) || shape[0] * (shape[1] ? shape[1] : 1) >= (int64_t)1 << 31)
    return fail(OXI_INVALID_ARGUMENT, "rotary: size exceeds the kernel limits");
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
  a.tokens = (uint32_t)shape[1];
  a.all = (uint32_t)(shape[0] * shape[1]);
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
  // A block's work: tokens and heads of ROWS units a thread, a load of each and
  // the end, or of one where there are too few for two blocks a CU: 8 units a
  // thread, loaded four at a time behind the stores before them, took 203 us
  // for (4, 4096, 32, 128) both ways, 4 at once 190, 2 179, 1 189.
  const int64_t wide = std::min<int64_t>(units, BS);
  const int64_t goal = (int64_t)a.all * a.heads * wide < (int64_t)ROWS * BS * 2 * cu_count() ? BS : ROWS * BS;
  int64_t heads = std::min<int64_t>(a.heads, std::max<int64_t>(1, goal / wide));
  int64_t tokens = std::max<int64_t>(1, goal / (heads * wide));
  tokens = std::min<int64_t>(std::min<int64_t>(tokens, MAX_TOKENS), a.half ? std::max(1, ANGLES / a.half) : MAX_TOKENS);
  tokens = std::min<int64_t>(tokens, a.all);
  a.block_tokens = (int)tokens;
  a.block_heads = (int)heads;
  a.units = (int)units;
  a.token_first = shape[1] > 1 && x_strides[1] < x_strides[2];
  const int64_t bx = ceil_div(a.all, tokens), by = ceil_div(a.heads, heads);
  if (!grid_fits(bx, BS) || by > 65535)
    return fail(OXI_INVALID_ARGUMENT, "rotary: size exceeds the kernel limits");
  const dim3 grid((unsigned)bx, (unsigned)by, (unsigned)ceil_div(units, BS));
  const size_t lds = sizeof(float) * 2 * (size_t)tokens * (size_t)a.half;
  const bool nts = nt_stream_stores(n * 4);
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

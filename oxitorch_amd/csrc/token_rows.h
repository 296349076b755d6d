// Rows of logits with one chosen class each, as the losses of post-training take
// them (token log-probabilities, policy and preference losses):
//
//   z = x/T, m = max x, t = (x - m) log2(e)/T, s = sum 2^t
//   logp = ln 2 t_a - ln s for the chosen class a,  H = ln s - ln 2 (sum 2^t t)/s
//   dx_j = (gl (d_ja - q_j) - gh q_j (ln q_j + H))/T,  q = 2^t/s
//
// for the gradients gl of logp and gh of H. The sums leave the chosen class out, so
// that 1 - q_a = rest/s and, where a has the largest logit, logp = -log1p(rest) keep
// their digits for a token that is all but certain; in 32 bits 1 - q_a would be 0
// or a multiple of 2^-24. Exponentials and a thread's sums of them are in 32 bits,
// relative to the maximum; what is formed of a row's sums is in 64.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "internal.h"
#include "launch_limits.h"
#include "row64.h"
#include "rowtile.h"

namespace oxi {

// Exponents below this count as this in the products 2^t t, where 2^t is 0: a class
// at -inf adds 0, not NaN.
constexpr float LEAST_T = -200.f;
constexpr double LOG_2 = 0.6931471805599453;

// log(1 + x) for x >= 0 (and NaN).
__device__ __forceinline__ double log1p64(double x) {
  if (!(x < 0.4)) return log64(1.0 + x);
  const double s = x / (2.0 + x), z = s * s;  // |s| < 0.167
  double p = 1.0 / 23;
#pragma unroll
  for (int k = 21; k > 0; k -= 2) p = fma(p, z, scalar(1.0 / k));
  return 2.0 * s * p;
}

// The rows of a call, and which of them count.
struct TokenRows {
  const float* x;
  const int64_t* ids;
  const float* weights;   // a row of weight 0 does not count; NULL: all do
  const int64_t* starts;  // rows outside [starts[0], starts[sequences]) do not; NULL: all do
  int64_t sequences;
  int64_t n;
  int c;
  float scale2;  // log2(e)/T
  double skew;   // by how much of itself scale2 is off
  double inv_t;
  int* guard;
  // where the parts' pass writes 0 for every row, and what rows that do not count keep; NULL: nowhere
  float *coef, *saved;

  // An id past the classes raises the guard and is padding.
  __device__ __forceinline__ bool counts(int64_t row, int64_t id) const {
    if (id >= c && (threadIdx.x & 15) == 0) atomicOr(guard, 1);
    return id >= 0 && id < c && (!weights || weights[row] != 0.f) &&
           (!starts || (row >= starts[0] && row < starts[sequences]));
  }
};

struct RowStats {
  double logp, entropy;
  float m, rest, total, off;  // off = entropy - ln total
};

// From the maximum m, the chosen logit xa and the sums over the other classes of 2^t
// and 2^t t. For values that are SUMMED over a sequence's tokens, what scale2 lost to its
// rounding, the same in every row, is taken back from logp to first order: d ln s = skew ln 2
// (sum 2^t t)/s. (A token's own ratio has it in its last bit; there it would cost registers:
// the policy loss of (8192, 32000) 325 us against 319.)
template <bool SUMMED>
__device__ __forceinline__ RowStats row_stats(float m, float xa, double rest, double et, const TokenRows& in) {
  const float ta = (xa - m) * in.scale2;
  const double ea = (double)__builtin_amdgcn_exp2f(ta);
  const double total = rest + ea;
  const double d = ((double)xa - (double)m) * in.inv_t;  // NaN where no class is left
  const double lt = d == 0.0 ? log1p64(rest) : log64(total);
  const double mean = (et + ea * (double)fmaxf(ta, LEAST_T)) / total;
  RowStats r;
  r.logp = d - (SUMMED ? lt - in.skew * (LOG_2 * mean) : lt);
  r.entropy = lt - LOG_2 * mean;
  r.m = m;
  r.rest = (float)rest;
  r.total = (float)total;
  r.off = (float)(-LOG_2 * mean);
  return r;
}

// What the backward needs of a row: its 4 floats of `saved`.
__device__ __forceinline__ void save_row(float* saved, int64_t row, const RowStats& r) {
  *reinterpret_cast<f4u*>(saved + 4 * row) = f4{r.m, r.rest, r.total, r.off};
}
__device__ __forceinline__ void save_nothing(float* saved, int64_t row) {
  *reinterpret_cast<f4u*>(saved + 4 * row) = f4{0.f, 0.f, 1.f, 0.f};
}

// v with component i at -inf.
__device__ __forceinline__ f4 drop(const f4& v, int i) {
  return f4{i == 0 ? NEG_INF : v.x, i == 1 ? NEG_INF : v.y, i == 2 ? NEG_INF : v.z, i == 3 ? NEG_INF : v.w};
}
__device__ __forceinline__ f4 put_at(const f4& v, int i, float a) {
  return f4{i == 0 ? a : v.x, i == 1 ? a : v.y, i == 2 ? a : v.z, i == 3 ? a : v.w};
}

// How a row of C classes lies: `head` classes, float4s, up to 3 classes more. The float4s
// begin at a 128-byte line (WHOLE; short rows: 16 bytes) or at 16 bytes.
template <bool WHOLE = true>
struct RowLay {
  static constexpr int EDGE = WHOLE ? 32 : 4;  // more than a head's classes
  int head, c4;
  __device__ __forceinline__ RowLay(const float* row, int C) : head(min(row_head(row, C), C)) {
    if (!WHOLE) head = min((int)(row_head(row, C) & 3), C);
    c4 = (C - head) >> 2;
  }
  // The class outside the float4s that thread t takes, or -1.
  __device__ __forceinline__ int edge(int t, int C) const {
    const int e = t < EDGE ? t : head + 4 * c4 + t - EDGE;
    return (t < EDGE ? t < head : t < EDGE + 3 && e < C) ? e : -1;
  }
  // The float4 of class a, or -1 outside of them; its component.
  __device__ __forceinline__ int slot(int a) const { return a >= head && a < head + 4 * c4 ? (a - head) >> 2 : -1; }
  __device__ __forceinline__ int component(int a) const { return (a - head) & 3; }
};

// Row and piece of block b of a launch of `pieces` blocks a row: a row's blocks on one XCD (blocks
// go round the 8 of them), so that what they all read of it misses one L2 once: (6288, 32000)
// of pairs 322 us against 343, log-probabilities of (8192, 32000) 165 against 170.
struct RowPiece {
  int64_t row;
  int piece;
  __device__ __forceinline__ RowPiece(uint32_t b, uint32_t rows, uint32_t pieces) {
    const uint32_t whole = rows & ~7u;
    if (b < whole * pieces) {
      const uint32_t i = b >> 3;
      row = (int64_t)(i / pieces * 8 + (b & 7));
      piece = (int)(i % pieces);
    } else {
      row = (int64_t)(b / pieces);
      piece = (int)(b % pieces);
    }
  }
};

// Rows cut into parts of PART_NT * PART_U float4s, a block each.
constexpr int PART_NT = 256, PART_U = 8;
inline int64_t row_parts(int64_t c) { return c > 0 ? ceil_div(c, (int64_t)PART_NT * PART_U * 4) : 1; }

// Maximum, sum and sum of 2^t t of each part, the chosen class left out; relative to
// the part's own maximum.
int launch_token_parts(const TokenRows& in, f4* parts, const char* what);

// The row of the parts mine[first], mine[first + step], .. as far as this lane adds them: maximum of all
// lanes in m; sums of this lane's.
__device__ __forceinline__ void join_parts(const f4* mine, int first, int step, int np, float m, float scale2, double& s,
                                           double& et) {
  s = et = 0.0;
  for (int p = first; p < np; p += step) {
    const f4 v = mine[p];
    if (v.y == 0.f) continue;  // nothing finite there
    const float d = (v.x - m) * scale2;
    const double f = (double)__builtin_amdgcn_exp2f(d);
    s += f * (double)v.y;
    et += f * ((double)v.z + (double)fmaxf(d, LEAST_T) * (double)v.y);
  }
}

// A row by one thread.
__device__ __forceinline__ RowStats joined_row(const TokenRows& in, const f4* mine, int np, float xa) {
  float m = xa;
  for (int p = 0; p < np; ++p) m = fmaxf(m, mine[p].x);
  double s, et;
  join_parts(mine, 0, 1, np, m, in.scale2, s, et);
  return row_stats<true>(m, xa, s, et, in);
}

// A wave a row: joins its parts; `op` writes what the row gives.
template <class Op>
__global__ __launch_bounds__(256) void token_join_k(const TokenRows in, const f4* __restrict__ parts, int np,
                                                    const Op op) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= in.n) return;
  const int64_t id = in.ids[row];
  if (!in.counts(row, id)) {
    if (lane == 0) op.skip(row);
    return;
  }
  const typename Op::Given given = op.load(row);
  const float xa = in.x[row * in.c + id];
  const f4* mine = parts + row * np;
  float m = xa;
  for (int p = lane; p < np; p += 64) m = fmaxf(m, mine[p].x);
  m = wave_max(m);
  double s, et;
  join_parts(mine, lane, 64, np, m, in.scale2, s, et);
  s = over_block<64, AddF64>(s, (double*)nullptr);
  et = over_block<64, AddF64>(et, (double*)nullptr);
  const RowStats r = row_stats<Op::SUMMED>(m, xa, s, et, in);
  op.finish(row, given, r, lane == 0);
}

// to[0] = the mean of `count` values, in 64 bits in a fixed order, by a block of MEAN_NT threads.
constexpr int MEAN_NT = 256;
struct MeanOf {
  const float* values;
  int64_t count;  // 0: nothing to do
  float* to;
  __device__ __forceinline__ void by_block() const {
    __shared__ double red[MEAN_NT / 64];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < count; i += MEAN_NT) s += (double)values[i];
    s = block_sum<MEAN_NT>(s, red);
    if (threadIdx.x == 0) to[0] = (float)(s / (double)count);
  }
};

// dx of the rows from their saved floats, for the gradients gl and gh (NULL: none) of
// their log-probabilities and entropies times gloss[0] (NULL: 1); and the mean, in a block more.
int launch_token_bwd(const float* x, const int64_t* ids, const float* saved, const float* gl, const float* gh,
                     const float* gloss, float* dx, int64_t n, int64_t c, float temperature, const char* what,
                     const MeanOf& mean = {});

// ---------------------------------------------------------------------------
// A row a group of RT threads (16 lanes, a wave, or a block), held in
// registers as NV float4s a thread: the logits cross HBM once for the loss and its
// gradient. Every thread works the row's few 64-bit formulas out by itself: from the
// first wave through LDS the kernel took 324 us against 316 at (8192, 32000) with a quarter padded.

// What a gradient at a class takes besides 2^t and t.
struct RowGrad {
  float alpha, beta, chosen;
  // For the gradients gl of logp and gh of the entropy.
  __device__ __forceinline__ RowGrad(const RowStats& r, float xa, float scale2, float inv_t, float gl, float gh) {
    const float a = gl * inv_t, b = gh * inv_t;
    alpha = -(a + b * r.off) / r.total;
    beta = -b * (float)LOG_2 / r.total;
    const float z = (xa - r.m) * scale2;
    const float q = __builtin_amdgcn_exp2f(z) / r.total;
    chosen = a * (r.rest / r.total) - (gh != 0.f ? b * q * fmaf((float)LOG_2, fmaxf(z, LEAST_T), r.off) : 0.f);
  }
};

// The row of block b: 16 neighbours go to one XCD (blocks go round the 8 of them), so that
// the lines of ids and of the rows' other numbers are read and written by one L2.
__device__ __forceinline__ int64_t row_of_block(uint32_t b, int64_t n) {
  const uint32_t g = b & ~127u;
  return (int64_t)g + 128 <= n ? (int64_t)(g + (b & 7) * 16 + ((b >> 3) & 15)) : (int64_t)b;
}

// Over a group of RT threads: 16 lanes, a wave or a block.
template <int RT, class R>
__device__ __forceinline__ typename R::T over_group(typename R::T v, typename R::T* slots) {
  if constexpr (RT >= 64) {
    return over_block<RT, R>(v, slots);
  } else {
    static_assert(RT == 16);
    v = R::op(v, R::template move<DPP_QUAD_XOR1>(v));
    v = R::op(v, R::template move<DPP_QUAD_XOR2>(v));
    v = R::op(v, R::template move<DPP_ROW_HALF_MIRROR>(v));
    return R::op(v, R::template move<DPP_ROW_MIRROR>(v));
  }
}

constexpr int rows_block(int rt) { return rt <= 64 ? 256 : rt; }
// Waves a SIMD: what the registers must allow, and at most, so that rows written as they
// are read do not crowd each other out.
constexpr int rows_waves(int rt, int nv) { return rt == 1024 && nv <= 8 ? 8 : 4; }
constexpr int rows_waves_most(bool grad, int nv) { return grad && nv >= 10 ? 4 : 8; }

template <int RT, int NV, bool GRAD, bool ENT, bool NTS, class Op>
__global__ __launch_bounds__(rows_block(RT)) __attribute__((amdgpu_waves_per_eu(rows_waves(RT, NV), rows_waves_most(GRAD, NV)))) void token_rows_k(
    const TokenRows in, const Op op, float* __restrict__ dx) {
  __shared__ __align__(8) float lds[RT > 64 ? 3 * (RT / 64) : 2];
  constexpr int ROWS = rows_block(RT) / RT;  // a block
  const int t = ROWS > 1 ? threadIdx.x & (RT - 1) : threadIdx.x;
  const int64_t row = ROWS > 1 ? (int64_t)blockIdx.x * ROWS + threadIdx.x / RT : row_of_block(blockIdx.x, in.n);
  if (ROWS > 1 && row >= in.n) return;
  const int C = in.c;
  const float* xr = in.x + row * C;
  float* dr = dx + row * C;
  const int64_t id64 = in.ids[row];
  const typename Op::Given given = op.load(row);
  const RowLay<(RT > 16)> lay(xr, C);
  auto put = [&](const f4& d, int c) {
    f4u* const p = reinterpret_cast<f4u*>(reinterpret_cast<char*>(dr + lay.head) + (uint32_t)c * 16u);
    if constexpr (NTS) __builtin_nontemporal_store(d, p);
    else *p = d;
  };
  const int e = lay.edge(t, C);
  if (!in.counts(row, id64)) {
    if (t == 0) op.skip(row);
    if constexpr (GRAD) {
#pragma unroll
      for (int q = 0; q < NV; ++q)
        if (q * RT + t < lay.c4) put(f4{0.f, 0.f, 0.f, 0.f}, q * RT + t);
      if (e >= 0) dr[e] = 0.f;
    }
    return;
  }
  const int id = (int)id64;
  const int at = lay.slot(id), comp = lay.component(id);
  const int at_q = at >= 0 ? at / RT : -1, at_t = at >= 0 ? at % RT : -1;
  const float xa = xr[id];
  f4 v[NV];
#pragma unroll
  for (int q = 0; q < NV; ++q)
    v[q] = ld_stream(reinterpret_cast<const f4*>(reinterpret_cast<const char*>(xr + lay.head) +
                                                 (uint32_t)min(q * RT + t, lay.c4 - 1) * 16u));
  float v1 = e >= 0 && e != id ? xr[e] : NEG_INF;
  float m = fmaxf(v1, xa);
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    if (q * RT + t >= lay.c4) v[q] = f4{NEG_INF, NEG_INF, NEG_INF, NEG_INF};
    if (q == at_q && t == at_t) v[q] = drop(v[q], comp);
    m = fmaxf(m, max4(v[q]));
  }
  m = over_group<RT, MaxF32>(m, lds);
  // With an entropy's gradient the registers keep t, else 2^t.
  float s = 0.f, et = 0.f;
  auto add = [&](float x) {
    const float z = (x - m) * in.scale2;
    const float p = __builtin_amdgcn_exp2f(z);
    s += p;
    et = fmaf(p, fmaxf(z, LEAST_T), et);
    return ENT ? z : p;
  };
#pragma unroll
  for (int q = 0; q < NV; ++q) v[q] = f4{add(v[q].x), add(v[q].y), add(v[q].z), add(v[q].w)};
  v1 = add(v1);
  const Two both = over_group<RT, Both<AddF32>>(Two{s, et}, reinterpret_cast<Two*>(lds + RT / 64));
  const RowStats r = row_stats<Op::SUMMED>(m, xa, (double)both.a, (double)both.b, in);
  const Two k = op.finish(row, given, r, t == 0);
  if constexpr (GRAD) {
    const RowGrad g(r, xa, in.scale2, (float)in.inv_t, k.a, ENT ? k.b : 0.f);
    auto grad = [&](float z) {
      // its exponential is formed again: held from the sums on, it would take the registers twice
      if constexpr (ENT) asm("" : "+v"(z));
      if constexpr (ENT) return __builtin_amdgcn_exp2f(z) * fmaf(g.beta, fmaxf(z, LEAST_T), g.alpha);
      else return z * g.alpha;
    };
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      if (q * RT + t >= lay.c4) continue;
      f4 d = f4{grad(v[q].x), grad(v[q].y), grad(v[q].z), grad(v[q].w)};
      if (q == at_q && t == at_t) d = put_at(d, comp, g.chosen);
      put(d, q * RT + t);
    }
    if (e >= 0) dr[e] = e == id ? g.chosen : grad(v1);
  }
}

// The row kernel for c classes: as few threads as hold the row; false past ROWS_MAX of
// them and under 8, where none does. Few rows too: 64 of 32000 are read in 7.5 us, by parts
// over more of the chip and their join in 7.7 (4 rows 7.0 and 6.5, 256 rows 9.7 and 11.4). The
// preference loss, whose pairs join parts without a launch of their own, pays for it: 92 rows of 32000
// in 2 pairs 18.5 us, by parts 17.7.
constexpr int ROWS_MAX = 32768;
template <bool GRAD, bool ENT, bool NTS, class Op>
bool launch_token_rows_as(const TokenRows& in, const Op& op, float* dx) {
  const int c4 = in.c / 4;  // at most
  if (in.c < 8 || in.c > ROWS_MAX) return false;
#define OXI_TR(RT, NV)                                                                                        \
  if (c4 <= RT * NV) {                                                                                        \
    token_rows_k<RT, NV, GRAD, ENT, NTS, Op>                                                                  \
        <<<dim3((unsigned)ceil_div(in.n, rows_block(RT) / RT)), dim3(rows_block(RT)), 0, stream()>>>(in, op, dx); \
    return true;                                                                                              \
  }
  OXI_TR(16, 4)
  OXI_TR(16, 8)
  OXI_TR(64, 4)
  OXI_TR(64, 8)
  OXI_TR(256, 4)
  OXI_TR(256, 8)
  OXI_TR(256, 12)
  OXI_TR(256, 16)
  if constexpr (!GRAD && !Op::SAME_BITS) {  // read alone, a block of fewer threads is faster
    OXI_TR(512, 10)
    OXI_TR(512, 12)
    OXI_TR(512, 14)
    OXI_TR(512, 16)
  } else {
    OXI_TR(1024, 5)
    OXI_TR(1024, 6)
    OXI_TR(1024, 7)
    OXI_TR(1024, 8)
  }
#undef OXI_TR
  return false;
}

// ---------------------------------------------------------------------------
// A row a cluster of blocks, each with a piece of it in registers (RT * NV float4s):
// rows that one block's registers do not hold. The blocks give each other their piece's
// maximum and sums by words of a value and a flag each, so that no order of memory
// accesses matters; the words are zeroed by a launch before. A block's row and piece go by a ticket that it takes as
// it starts: a block waits only for those of its own row, which have started or take
// the next tickets, and the rows before finish without it, so every wait ends; one that does not, as where
// two calls share a workspace, gives up: the guard flag (bit 8), and NaN in what that block writes of its row.
// (1024, 131072) with an entropy term 190 us, 5.4 TB/s; parts, their join and the
// backward's pass 244. (4096, 50257) on two blocks 280, on one of 1024 threads 308. For few shorter rows, (64, 32000) on 4 blocks each, the ticket
// and the words cost what the other CUs gain: 11.0 us against 10.2 on one block.
constexpr int CLUSTER_RT = 512, CLUSTER_MOST = 16;
struct Cluster {
  uint64_t* words;  // 3 a block
  uint32_t* ticket;
  int blocks;  // a row
  int spin_limit;
};
inline int64_t cluster_bytes(int64_t n, int blocks) { return 64 + n * blocks * 3 * (int64_t)sizeof(uint64_t); }
// words and ticket zeroed, in `at`
Cluster start_cluster(void* at, int64_t n, int blocks);

constexpr uint64_t WORD_SET = (uint64_t)1 << 32;
__device__ __forceinline__ void give_word(uint64_t* p, float v) {
  __hip_atomic_store(p, WORD_SET | __float_as_uint(v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// The word once it is set; NaN after spin_limit polls more (a negative limit: at once).
__device__ __forceinline__ float take_word(const uint64_t* p, int spin_limit, int* guard) {
  for (int spins = 0; spins <= spin_limit; ++spins) {
    const uint64_t v = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (v & WORD_SET) return __uint_as_float((uint32_t)v);
    __builtin_amdgcn_s_sleep(1);
  }
  atomicOr(guard, 8);
  return __builtin_nanf("");
}

template <int NV, bool GRAD, bool ENT, bool NTS, class Op>
__global__ __launch_bounds__(CLUSTER_RT) __attribute__((amdgpu_waves_per_eu(4, 4))) void token_cluster_k(
    const TokenRows in, const Op op, float* __restrict__ dx, const Cluster cl) {
  constexpr int RT = CLUSTER_RT;
  __shared__ __align__(8) float lds[3 * (RT / 64)];
  __shared__ float from[3 * CLUSTER_MOST];
  __shared__ uint32_t ticket;
  const int t = threadIdx.x;
  if (t == 0) ticket = atomicAdd(cl.ticket, 1u);
  __syncthreads();
  const uint32_t b = __builtin_amdgcn_readfirstlane(ticket);
  const int64_t row = b / (unsigned)cl.blocks;
  if (row >= in.n) {  // another call has taken tickets from this workspace: there is no such row
    if (t == 0) atomicOr(in.guard, 8);
    return;
  }
  const int piece = (int)(b % (unsigned)cl.blocks);
  const int C = in.c;
  const float* xr = in.x + row * C;
  float* dr = dx + row * C;
  const int64_t id64 = in.ids[row];
  const RowLay<> lay(xr, C);
  const int c0 = piece * (RT * NV) + t;
  auto put = [&](const f4& d, int c) {
    f4u* const p = reinterpret_cast<f4u*>(dr + lay.head) + c;
    if constexpr (NTS) __builtin_nontemporal_store(d, p);
    else *p = d;
  };
  const int e = piece == 0 ? lay.edge(t, C) : -1;
  const bool lead = piece == 0 && t == 0;
  uint64_t* const words = cl.words + 3 * cl.blocks * row;
  if (!in.counts(row, id64)) {
    if (t < 3) give_word(words + 3 * piece + t, 0.f);  // no wait hangs on all blocks seeing the same
    if (lead) op.skip(row);
    if constexpr (GRAD) {
#pragma unroll
      for (int q = 0; q < NV; ++q)
        if (c0 + q * RT < lay.c4) put(f4{0.f, 0.f, 0.f, 0.f}, c0 + q * RT);
      if (e >= 0) dr[e] = 0.f;
    }
    return;
  }
  const int id = (int)id64;
  const int at = lay.slot(id), comp = lay.component(id);
  const float xa = xr[id];
  f4 v[NV];
#pragma unroll
  for (int q = 0; q < NV; ++q) v[q] = ld_stream(reinterpret_cast<const f4*>(xr + lay.head) + min(c0 + q * RT, lay.c4 - 1));
  float v1 = e >= 0 && e != id ? xr[e] : NEG_INF;
  float own = v1;
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    if (c0 + q * RT >= lay.c4) v[q] = f4{NEG_INF, NEG_INF, NEG_INF, NEG_INF};
    if (c0 + q * RT == at) v[q] = drop(v[q], comp);
    own = fmaxf(own, max4(v[q]));
  }
  own = over_block<RT, MaxF32>(own, lds);
  const float shift = own == NEG_INF ? 0.f : own;
  // With an entropy's gradient the registers keep t relative to the piece's maximum, else 2^t.
  float s = 0.f, et = 0.f;
  auto add = [&](float x) {
    const float z = (x - shift) * in.scale2;
    const float p = __builtin_amdgcn_exp2f(z);
    s += p;
    et = fmaf(p, fmaxf(z, LEAST_T), et);
    return ENT ? z : p;
  };
#pragma unroll
  for (int q = 0; q < NV; ++q) v[q] = f4{add(v[q].x), add(v[q].y), add(v[q].z), add(v[q].w)};
  v1 = add(v1);
  const Two both = over_block<RT, Both<AddF32>>(Two{s, et}, reinterpret_cast<Two*>(lds + RT / 64));
  if (t < 3) give_word(words + 3 * piece + t, t == 0 ? own : t == 1 ? both.a : both.b);
  if (t < 3 * cl.blocks) from[t] = take_word(words + t, cl.spin_limit, in.guard);
  __syncthreads();
  float m = xa;
  for (int k = 0; k < cl.blocks; ++k) m = fmaxf(m, from[3 * k]);
  double rest = 0.0, mean = 0.0;
  for (int k = 0; k < cl.blocks; ++k) {
    if (from[3 * k + 1] == 0.f) continue;  // nothing finite there
    const float d = (from[3 * k] - m) * in.scale2;
    const double f = (double)__builtin_amdgcn_exp2f(d);
    rest += f * (double)from[3 * k + 1];
    mean += f * ((double)from[3 * k + 2] + (double)fmaxf(d, LEAST_T) * (double)from[3 * k + 1]);
  }
  const RowStats r = row_stats<Op::SUMMED>(m, xa, rest, mean, in);
  const Two k = op.finish(row, op.load(row), r, lead);
  if constexpr (GRAD) {
    const RowGrad g(r, xa, in.scale2, (float)in.inv_t, k.a, ENT ? k.b : 0.f);
    // The piece's t from the row's, never above 0: a piece without a finite logit has a shift of 0, which
    // may lie far over m, and its 2^t of 0 must not meet an infinite factor.
    const float up = fminf((shift - m) * in.scale2, 0.f);
    const float alpha = ENT ? g.alpha : g.alpha * __builtin_amdgcn_exp2f(up);
    auto grad = [&](float z) {
      if constexpr (ENT) {
        asm("" : "+v"(z));  // its exponential is formed again, not held
        z += up;
        return __builtin_amdgcn_exp2f(z) * fmaf(g.beta, fmaxf(z, LEAST_T), alpha);
      } else {
        return z * alpha;
      }
    };
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      if (c0 + q * RT >= lay.c4) continue;
      f4 d = f4{grad(v[q].x), grad(v[q].y), grad(v[q].z), grad(v[q].w)};
      if (c0 + q * RT == at) d = put_at(d, comp, g.chosen);
      put(d, c0 + q * RT);
    }
    if (e >= 0) dr[e] = e == id ? g.chosen : grad(v1);
  }
}

// The blocks a row of c classes: as few as hold it; 0 where one block does, or more
// than CLUSTER_MOST would be needed.
constexpr int CLUSTER_NV = 16;
inline int cluster_blocks(int64_t c) {
  const int64_t blocks = ceil_div(c, (int64_t)CLUSTER_RT * CLUSTER_NV * 4);
  return c > ROWS_MAX && blocks <= CLUSTER_MOST ? (int)blocks : 0;
}

template <bool GRAD, bool ENT, bool NTS, class Op>
bool launch_token_cluster(const TokenRows& in, const Op& op, float* dx, void* workspace) {
  const int blocks = cluster_blocks(in.c);
  if (!blocks || !grid_fits(in.n * blocks, CLUSTER_RT)) return false;
  const Cluster cl = start_cluster(workspace, in.n, blocks);
  const dim3 grid((unsigned)(in.n * blocks));
#define OXI_TC(NV)                                                                                           \
  if ((int64_t)blocks * CLUSTER_RT * NV * 4 >= in.c) {                                                       \
    token_cluster_k<NV, GRAD, ENT, NTS, Op><<<grid, dim3(CLUSTER_RT), 0, stream()>>>(in, op, dx, cl);        \
    return true;                                                                                             \
  }
  OXI_TC(9)
  OXI_TC(10)
  OXI_TC(12)
  OXI_TC(14)
  OXI_TC(CLUSTER_NV)
#undef OXI_TC
  return false;
}

// Whether sizes and temperature can be taken; 0 or an error's code.
int check_token_rows(const char* what, int64_t n, int64_t c, float temperature);
TokenRows token_rows(const float* x, const int64_t* ids, int64_t n, int64_t c, float temperature);

// Bytes of the parts of n rows.
inline int64_t token_parts_bytes(int64_t n, int64_t c) { return n * row_parts(c) * (int64_t)sizeof(f4); }

// The rows' results without a gradient: by parts, or, where it takes them, by the row kernel.
template <class Op>
int token_rows_by_parts(const TokenRows& in, f4* parts, const Op& op, const char* what) {
  if (int rc = launch_token_parts(in, parts, what)) return rc;
  token_join_k<Op><<<dim3((unsigned)ceil_div(in.n, 4)), dim3(256), 0, stream()>>>(in, parts, (int)row_parts(in.c), op);
  return check_launch(what);
}
template <class Op>
int token_rows_read(const TokenRows& in, f4* parts, const Op& op, const char* what) {
  return launch_token_rows_as<false, false, false>(in, op, nullptr) ? check_launch(what)
                                                                    : token_rows_by_parts(in, parts, op, what);
}

}  // namespace oxi

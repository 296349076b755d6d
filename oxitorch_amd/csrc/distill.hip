// Distillation from a teacher's top logits for gfx950: the divergence of a
// student's softmax over c classes from a teacher known by its k best entries a
// row, with its gradient.
//
//   z = x/T, q = exp(z - lse), p the teacher's entries (softmaxed over the row's
//   k, or given the teacher's log-sum-exp, with pr = 1 - sum p left over)
//   row = sum p (log p - log q[id]) + pr (log pr - log qr)
//   dx  = T/divisor (q - p) at the entries, T/divisor q (1 - pr/qr) elsewhere
//         (sum p + pr = 1: not q (sum p + pr) for q)
//
// The k entries of a row are worked out in 64 bits by the block that owns the
// row: a student near its teacher has a small loss of terms that cancel. With
// the rest's term both sides' masses are 1, and the row is summed as
// q - p + p log(p/q), each of which is >= 0, so that an error of lse enters
// squared. qr is a sum over the classes that are not listed, never 1 minus the
// listed, and those have a maximum of their own: s = softmax over them and log qr are
// there where qr itself is below the smallest float, and their gradient is
// T/divisor s (qr - pr).
#include <cmath>

#include "internal.h"
#include "launch_limits.h"
#include "row64.h"
#include "rowtile.h"

namespace oxi {
namespace {

constexpr int NT = 256;
// Classes that one bitmap of listed ids covers (8 KB of LDS); longer rows are
// walked in stretches of it.
constexpr int STRETCH = 65536;

struct DistillArgs {
  const float* x;
  const int64_t* ids;
  const float* top;
  const float* top_lse;
  float* row_loss;
  float* lse;
  float* rest;
  float* dx;
  int64_t n;
  int c, k;
  float inv_t;
  double t;  // temperature
  float divisor;
  const float* count;  // the divisor if it lies on the device, else NULL
  const float* gloss;  // the upstream gradient, NULL for 1
  int* guard;

  __device__ __forceinline__ float divided_by() const { return count ? count[0] : divisor; }
  __device__ __forceinline__ float upstream() const { return gloss ? gloss[0] : 1.f; }
  __device__ __forceinline__ float grad_scale(float over, float up) const { return (float)t / over * up; }
};

// A row's teacher entries in LDS: class ids (-1: padding, or an id that an
// earlier entry has, then in `dup`), probabilities and their logarithms.
struct Teacher {
  double* p;
  double* lp;
  int* id;
  int* dup;
  int* seen;   // a hash table of the ids, seen_slots(k) of them
  bool twice;  // whether any id is given twice
};
// A power of two, at least twice the entries: a probe always ends at a free slot.
constexpr int seen_slots(int64_t k) {
  int n = 2;
  while (n < 2 * k) n *= 2;
  return n;
}
constexpr size_t teacher_bytes(int64_t k) {
  return (size_t)k * (2 * sizeof(double) + 2 * sizeof(int)) + (size_t)seen_slots(k) * sizeof(int);
}

__device__ __forceinline__ Teacher teacher_at(double* lds, int k) {
  Teacher a;
  a.p = lds;
  a.lp = lds + k;
  a.id = reinterpret_cast<int*>(lds + 2 * k);
  a.dup = a.id + k;
  a.seen = a.dup + k;
  return a;
}

// Fills `a` with the row's entries; returns the sum of p, and in `some` whether
// there is any entry. All threads of the block; the entries are published. Ids
// given twice are rare: the entries' order is looked up only where the hash table
// met one.
template <int N>
__device__ __forceinline__ double load_teacher(const DistillArgs& g, int64_t row, Teacher& a, double* red,
                                               bool& some) {
  const int64_t* ids = g.ids + row * g.k;
  const float* top = g.top + row * g.k;
  float* redf = reinterpret_cast<float*>(red);
  float tm = NEG_INF;
  int any = 0;
  const int slots = seen_slots(g.k);
  for (int i = threadIdx.x; i < slots; i += N) a.seen[i] = -1;
  for (int j = threadIdx.x; j < g.k; j += N) {
    const int64_t id = ids[j];
    const float v = top[j];
    if (id >= g.c) atomicOr(g.guard, 1);
    const bool there = id >= 0 && id < g.c && v != NEG_INF;
    a.id[j] = there ? (int)id : -1;
    a.lp[j] = (double)v;
    if (there) {
      tm = fmaxf(tm, v);
      any = 1;
    }
  }
  some = __syncthreads_or(any) != 0;
  tm = group_max<N>(tm, redf);
  int met = 0;
  double s = 0.0;
  for (int j = threadIdx.x; j < g.k; j += N) {
    const bool there = a.id[j] >= 0;
    const double v = a.lp[j];
    const double l = g.top_lse ? v / g.t - (double)g.top_lse[row] : (v - (double)tm) / g.t;
    const double p = there ? exp64(l) : 0.0;
    a.lp[j] = l;
    a.p[j] = p;
    s += p;
    a.dup[j] = -1;
    if (there) {
      const int id = a.id[j];
      for (int h = (int)((uint32_t)id * 2654435761u >> 16) & (slots - 1);; h = (h + 1) & (slots - 1)) {
        const int old = atomicCAS(a.seen + h, -1, id);
        if (old == -1) break;
        if (old == id) {
          met = 1;
          break;
        }
      }
    }
  }
  s = block_sum<N>(s, red);
  a.twice = __syncthreads_or(met) != 0;
  if (a.twice) {
    for (int j = threadIdx.x; j < g.k; j += N)
      if (a.id[j] >= 0)
        for (int i = 0; i < j && a.dup[j] < 0; ++i)
          if (a.id[i] == a.id[j]) a.dup[j] = i;
  }
  if (!g.top_lse && some) {  // divide by the sum
    const double ls = log64(s);
    for (int j = threadIdx.x; j < g.k; j += N) {
      a.p[j] = a.p[j] / s;
      a.lp[j] -= ls;
    }
    s = 1.0;
  }
  __syncthreads();
  return s;
}

// An entry's share of the row's sum, lq the logarithm of the student's
// probability of it.
__device__ __forceinline__ double entry_term(double p, double lp, double lq, bool tail, bool dup) {
  const double d = lq - lp;  // log(q / p)
  if (!tail) return p > 0.0 || p != p ? -p * d : 0.0;
  if (dup) return p > 0.0 || p != p ? -p * d - p : 0.0;
  return p > 0.0 || p != p ? p * exp_rest(d) : exp64(lq);
}

// What entries of sum psum leave to the other classes.
__device__ __forceinline__ double rest_of(double psum) { return psum < 1.0 ? 1.0 - psum : psum != psum ? psum : 0.0; }

// That, given whether the student's mass there is below 2^-126, as of masked logits
// (-inf or the lowest float): a rest of the size that rounding leaves in a log-sum-exp
// worked out in 32 bits (4 steps of it and of 1) is none then. Its loss would be that
// rounding times their distance.
template <class F>
__device__ __forceinline__ F rest_beside(F pr, bool masked, float top_lse) {
  return masked && pr <= (F)0x1p-22 * ((F)1 + (F)fabsf(top_lse)) ? (F)0 : pr;
}

// The rest's share, lr the logarithm of the student's mass there, with what the
// masses as rounded lack of 1.
__device__ __forceinline__ double rest_term(double psum, double lr, float top_lse) {
  const double pr = rest_beside(rest_of(psum), lr < -126 * 0.6931471805599453, top_lse);
  return (pr > 0.0 || pr != pr ? pr * exp_rest(lr - log64(pr)) : exp64(lr)) + ((psum + pr) - 1.0);
}

// A row's results: its loss, its log-sum-exp and the logarithm lr of the student's
// mass at the classes not listed, from the log-sum-exp as stored.
__device__ __forceinline__ void write_row(const DistillArgs& g, int64_t row, bool some, double terms, double lse,
                                          double lr) {
  const float l = (float)lse;
  g.row_loss[row] = some ? (float)(g.t * g.t * terms) : 0.f;
  g.lse[row] = l;
  g.rest[row] = (float)(lr + (lse - (double)l));
}

// qr - pr, from the masses ql and psum of the listed classes where those are the smaller.
template <class F>
__device__ __forceinline__ F rest_excess(F psum, F ql, F qr, F pr, float top_lse) {
  return psum < (F)0.5 ? psum - ql : qr - rest_beside(pr, qr < (F)0x1p-126, top_lse);
}

// The gradient at the row's entries, after the block has written the row as if
// none were listed.
template <int N, class Q>
__device__ __forceinline__ void write_entries(const DistillArgs& g, int64_t row, const Teacher& a, float gscale, Q q) {
  __syncthreads();
  float* dr = g.dx + row * g.c;
  for (int j = threadIdx.x; j < g.k; j += N) {
    const int id = a.id[j];
    if (id < 0 || a.dup[j] >= 0) continue;
    double p = a.p[j];
    if (a.twice)
      for (int i = j + 1; i < g.k; ++i)
        if (a.dup[i] == j) p += a.p[i];
    dr[id] = (float)(q(j, id) - p) * gscale;
  }
}

// Sets the bits of the row's listed classes in [c0, c0 + STRETCH).
template <int N>
__device__ __forceinline__ void mark_listed(const Teacher& a, int k, int c0, uint32_t* bits) {
  __syncthreads();
  for (int i = threadIdx.x; i < STRETCH / 32; i += N) bits[i] = 0;
  __syncthreads();
  for (int j = threadIdx.x; j < k; j += N) {
    const int e = a.id[j] - c0;
    if (a.id[j] >= 0 && e >= 0 && e < STRETCH) atomicOr(bits + (e >> 5), 1u << (e & 31));
  }
  __syncthreads();
}

// A block a row of any length, which it walks twice, the first time with a running
// maximum: under 8 classes, and past STREAM_MAX of them, where the row comes from
// HBM each time.
__global__ __launch_bounds__(NT) void distill_loop_k(const DistillArgs g) {
  extern __shared__ __align__(16) double dyn[];
  __shared__ double red[NT / 64];
  __shared__ uint32_t bits[STRETCH / 32];
  Teacher a = teacher_at(dyn, g.k);
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  const bool tail = g.top_lse != nullptr;
  const float* xr = g.x + row * g.c;
  bool some;
  const double psum = load_teacher<NT>(g, row, a, red, some);
  // maximum and sum over the classes not listed (without the rest's term over all)
  float mr = NEG_INF;
  double sum = 0.0;
  for (int c0 = 0; c0 < g.c; c0 += STRETCH) {
    if (tail) mark_listed<NT>(a, g.k, c0, bits);
    const int end = min(g.c - c0, STRETCH);
    for (int c = t; c < end; c += NT) {
      if (tail && (bits[c >> 5] >> (c & 31) & 1)) continue;
      const float v = xr[c0 + c];
      if (v > mr) {
        sum *= expf((mr - v) * g.inv_t);
        mr = v;
      }
      sum += expf((v - (mr == NEG_INF ? 0.f : mr)) * g.inv_t);
    }
  }
  const float own = mr;
  mr = group_max<NT>(mr, reinterpret_cast<float*>(red));
  if (own != NEG_INF) sum *= expf((own - mr) * g.inv_t);
  sum = block_sum<NT>(sum, red);
  // and the listed ones
  float ml = NEG_INF;
  double listed = 0.0;
  if (tail) {
    for (int j = t; j < g.k; j += NT)
      if (a.id[j] >= 0) ml = fmaxf(ml, xr[a.id[j]]);
    ml = group_max<NT>(ml, reinterpret_cast<float*>(red));
  }
  const float m = fmaxf(mr, ml);
  if (tail) {
    for (int j = t; j < g.k; j += NT)
      if (a.id[j] >= 0 && a.dup[j] < 0) listed += expf((xr[a.id[j]] - m) * g.inv_t);
    listed = block_sum<NT>(listed, red);
  }
  const double below = ((double)mr - (double)m) / g.t;  // the rest's maximum from the row's
  const double total = tail ? sum * exp64(below) + listed : sum;
  const double lt = log64(total), lr = log64(sum) + below - lt;
  if (g.row_loss) {
    double s = 0.0;
    for (int j = t; j < g.k; j += NT)
      if (a.id[j] >= 0)
        s += entry_term(a.p[j], a.lp[j], ((double)xr[a.id[j]] - (double)m) / g.t - lt, tail, a.dup[j] >= 0);
    s = block_sum<NT>(s, red);
    if (tail && some) s += rest_term(psum, lr, g.top_lse[row]);
    if (t == 0) write_row(g, row, some, s, (double)m / g.t + lt, tail ? lr : 0.0);
  }
  if (!g.dx) return;
  const float gscale = g.grad_scale(g.divided_by(), g.upstream());
  double share = tail ? rest_excess(psum, listed / total, exp64(lr), rest_of(psum), g.top_lse[row]) : 1.0;
  share = sum > 0.0 || sum != sum ? share / sum : 0.0;
  const float scale = (float)share * gscale, shift = tail && mr == NEG_INF ? 0.f : mr;
  float* dr = g.dx + row * g.c;
  for (int c = t; c < g.c; c += NT) dr[c] = some ? expf((xr[c] - shift) * g.inv_t) * scale : 0.f;
  write_entries<NT>(g, row, a, gscale,
                    [&](int, int id) { return (double)expf((xr[id] - m) * g.inv_t) / total; });
}

// ---------------------------------------------------------------------------
// A row a block: RT * NV float4s held in registers, so the logits cross HBM once
// for the loss and its gradient. The float4s begin at a row's first 128-byte line;
// the classes before and after them go a float to a thread. Exponentials are exp2
// of (x - m) * (log2(e)/T). With the rest's term the listed classes are taken out
// of the registers (an exponential of 0) by a bitmap in LDS, m is the maximum of the
// others, and the entries' threads add the listed ones' own few. The block's stores
// write the row as if nothing were listed; the entries' values go over that after a
// barrier.
//
// HBM bounds it: (8192, 32000) with 64 entries and the rest 354-364 us, 5.8-6.1 TB/s;
// (4096, 50257) 285 us, 5.8 TB/s; 64 rows of 32000 10 us, a row a CU. The entries
// are worked out in float64 before the row is reduced and their terms after it is
// stored, from LDS, so that the registers of that code do not add to the row's: at
// most 128 a lane, two blocks of 512 x 16 a CU. The row's loads go out before the
// entries' work in those (with the rest's term (8192, 32000) 364 us, 376 behind
// it), and behind it where a block has the CU to itself ((4096, 50257) 301 us
// before it, 288 behind) or four share it ((4096, 8192) with the rest's term 56
// and 53).
//
// The backward for an upstream scalar is the same pass without the loss (no
// row_loss): (8192, 32000) 359-368 us. From a log-sum-exp rounded to a float every
// probability of a row would be off by up to |lse| 2^-24 of itself, 6e-4 at logits near
// 10^4; here its error goes by the distance from the maximum. Rows that no registers
// hold take the two floats lse and rest instead of a pass for their sums ((1500, 100001)
// 229 us, 261 with it).
//
// NV = 0: longer rows, streamed twice, the first time with a running maximum. Two
// blocks fit a CU, so that up to 512 rows are between their passes: 205 MB of 100001
// classes, which the Infinity Cache (256 MB) holds, but 268 of 131072 and 614 of 300000.
// (1500, 100001) 261 us, 4.6 TB/s of the bytes that one pass needs; (2048, 128256)
// 447 us, 4.7; (1024, 200000) 372, 4.4; (800, 300000) 505, 3.8. With one block a CU 253,
// 445, 359 and 450, and the loss alone of (1500, 100001) 116 where two take 103.
constexpr int STREAM_U = 4;         // float4s in flight a thread
constexpr int STREAM_MAX = 300000;  // classes whose bitmap fits in LDS beside 1024 entries

// Waves a SIMD that the registers must allow: 4 with 128 a lane, 8 with 64; and at
// most, so that rows written as they are read do not crowd each other out: a third
// block of 512 threads a CU took (16384, 16640) with the rest's term from 366 to 400 us,
// a fifth of 256 (8192, 12000) from 136 to 144.
constexpr int rows_waves(int nv) { return nv ? 4 : 8; }
constexpr int rows_waves_most(bool grad, int nv) { return grad && nv >= 10 ? 4 : 8; }

// Words of the bitmap of C classes, which starts up to 32 bits in.
constexpr int bitmap_words(int C) { return (C + 32 + 31) / 32 + 1; }

// v with the classes of set bits at -inf.
__device__ __forceinline__ f4 without(const f4& v, uint32_t bits) {
  return f4{bits & 1 ? NEG_INF : v.x, bits & 2 ? NEG_INF : v.y, bits & 4 ? NEG_INF : v.z, bits & 8 ? NEG_INF : v.w};
}

template <int RT, int NV, bool GRAD, bool TAIL, bool NTS>
__global__ __launch_bounds__(RT)
    __attribute__((amdgpu_waves_per_eu(rows_waves(NV), rows_waves_most(GRAD, NV)))) void distill_rows_k(
        const DistillArgs g, const float scale2) {
  __shared__ double red[RT / 64], psum_at;
  __shared__ __align__(8) float lds[4 * (RT / 64)];
  __shared__ int twice;
  // k probabilities, k logarithms of them, k ids (-1: padding, -2 - id: an id
  // that an earlier entry has), the student's logits there, a bit a class
  extern __shared__ __align__(16) double dyn[];
  double* const ep = dyn;
  double* const elp = dyn + g.k;
  int* const eid = reinterpret_cast<int*>(dyn + 2 * g.k);
  float* const ex = reinterpret_cast<float*>(eid + g.k);
  uint32_t* const bits = reinterpret_cast<uint32_t*>(ex + g.k);
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int C = g.c;
  const float* xr = g.x + row * C;
  // the row's classes before its first 16-byte address, and its float4s from there
  const int head = row_head(xr, C);
  const int c4 = (C - head) >> 2;
  // float4 c at a 32-bit byte offset from a uniform address: one register an
  // access, not two
  auto x4 = [&](int c) -> const f4* {
    return reinterpret_cast<const f4*>(reinterpret_cast<const char*>(xr + head) + (uint32_t)c * 16u);
  };
  // used after the row's sums: nothing waits for them before (a wait here, 366
  // to 393 us backward at (16384, 16640))
  const float up = GRAD ? g.upstream() : 1.f, over = GRAD ? g.divided_by() : 1.f;
  // the entries' loads go first (a thread's first one; the rest of long lists
  // later): a wait for them leaves the row's in flight, if those are
  const int64_t id0 = t < g.k ? g.ids[row * g.k + t] : -1;
  const float top0 = t < g.k ? g.top[row * g.k + t] : 0.f;
  const float tlse = TAIL ? g.top_lse[row] : 0.f;
  // one of the up to 31 classes before the float4s, or the 3 after them
  const int e1 = t < 32 ? t : head + 4 * c4 + t - 32;
  const bool has1 = t < 32 ? t < head : t < 35 && e1 < C;
  float v1 = has1 ? xr[e1] : NEG_INF;
  f4 v[NV ? NV : 1];
  auto load_row = [&]() {
#pragma unroll
    for (int q = 0; q < NV; ++q) v[q] = ld_stream(x4(min(q * RT + t, c4 - 1)));
  };
  if constexpr (RT == 512) load_row();
  for (int i = t; i < bitmap_words(C); i += RT) bits[i] = 0;
  if (t == 0) twice = 0;
  // the student's logit at this thread's first entry: waited for after the
  // entries' arithmetic
  const float x0 = id0 >= 0 && id0 < C ? xr[id0] : NEG_INF;
  bool some;
  float psumf = 0.f, prf = 0.f;  // the entries' mass, and what they leave
  {
    // the thread's first entry in registers, the others of a long list through LDS
    const bool there0 = id0 >= 0 && id0 < C && top0 != NEG_INF;
    bool any = there0;
    float tm = there0 ? top0 : NEG_INF;
    if (id0 >= C) atomicOr(g.guard, 1);
    if (t < g.k) eid[t] = there0 ? (int)id0 : -1;
#pragma unroll 1
    for (int j = t + RT; j < g.k; j += RT) {
      const int64_t id = g.ids[row * g.k + j];
      const float top = g.top[row * g.k + j];
      const bool there = id >= 0 && id < C && top != NEG_INF;
      if (id >= C) atomicOr(g.guard, 1);
      eid[j] = there ? (int)id : -1;
      elp[j] = (double)top;
      any |= there;
      tm = fmaxf(tm, there ? top : NEG_INF);
    }
    some = __syncthreads_or(any) != 0;  // and the bitmap is clear
    if constexpr (!TAIL) tm = over_block<RT, MaxF32>(tm, lds);
    auto mark = [&](int id) {
      const int at = id + 32 - head;  // float4 c has the four bits from 32 + 4 c
      const uint32_t bit = 1u << (at & 31);
      if (atomicOr(bits + (at >> 5), bit) & bit) twice = 1;
    };
    auto log_of = [&](double top) { return TAIL ? top / g.t - (double)tlse : (top - (double)tm) / g.t; };
    if (there0) mark((int)id0);
    double l0 = log_of((double)top0);
    double p0 = there0 ? exp64(l0) : 0.0;
    double psum = p0;
#pragma unroll 1
    for (int j = t + RT; j < g.k; j += RT) {
      if (eid[j] >= 0) mark(eid[j]);
      const double l = log_of(elp[j]);
      const double p = eid[j] >= 0 ? exp64(l) : 0.0;
      elp[j] = l;
      ep[j] = p;
      psum += p;
    }
    psum = block_sum<RT>(psum, red);  // its barriers publish the bitmap and the entries
    if constexpr (!TAIL) {
      const double ls = log64(psum);
      p0 = there0 ? p0 / psum : 0.0;
      l0 -= ls;
#pragma unroll 1
      for (int j = t + RT; j < g.k; j += RT) {
        ep[j] = eid[j] >= 0 ? ep[j] / psum : 0.0;
        elp[j] -= ls;
      }
    }
    if (t < g.k) {
      ep[t] = p0;
      elp[t] = l0;
    }
    if (twice) {  // ids given twice: rare, so their order is looked up only then
      // (an entry's code changes once, from id to -2 - id, and either names the id)
#pragma unroll 1
      for (int j = t; j < g.k; j += RT) {
        const int id = eid[j];
        bool dup = false;
        for (int i = 0; i < j && !dup; ++i) dup = id >= 0 && (eid[i] == id || eid[i] == -2 - id);
        if (dup) eid[j] = -2 - id;
      }
      __syncthreads();
    }
    if (t < g.k) ex[t] = there0 ? x0 : NEG_INF;
#pragma unroll 1
    for (int j = t + RT; j < g.k; j += RT) ex[j] = eid[j] == -1 ? NEG_INF : xr[eid[j] < 0 ? -2 - eid[j] : eid[j]];
    if (t == 0) psum_at = psum;
    psumf = uniform((float)psum);
    prf = uniform((float)rest_of(psum));
  }
  if constexpr (RT != 512) load_row();
  auto listed = [&](int c) -> uint32_t { return TAIL ? bits[(c >> 3) + 1] >> ((c & 7) * 4) & 15u : 0u; };
  if (TAIL && has1 && (bits[(e1 + 32 - head) >> 5] >> ((e1 + 32 - head) & 31) & 1u)) v1 = NEG_INF;
  // The maximum mr and the sum of exponentials of the classes not listed (without
  // the rest's term: of all), then the row's maximum m and its sum `total`.
  float mr = NEG_INF, m, s = 0.f;
  bool known = false;
  auto maxima = [&]() {
    if (!known) mr = fmaxf(mr, v1);
    if constexpr (TAIL) {
      float ml = NEG_INF;
#pragma unroll 1
      for (int j = t; j < g.k; j += RT) ml = fmaxf(ml, ex[j]);
      const Two both = over_block<RT, Both<MaxF32>>(Two{mr, ml}, reinterpret_cast<Two*>(lds));
      mr = both.a;
      m = fmaxf(both.a, both.b);
    } else {
      m = mr = over_block<RT, MaxF32>(mr, lds + RT / 64);
    }
  };
  // what logits are taken relative to; with nothing finite there, their exponentials are 0
  auto shift_of = [&](float top) { return TAIL && top == NEG_INF ? 0.f : top; };
  if constexpr (NV > 0) {
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      const int c = q * RT + t;
      v[q] = without(v[q], c < c4 ? listed(c) : 15u);
      mr = fmaxf(mr, max4(v[q]));
    }
    maxima();
    const float shift = shift_of(mr);
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      v[q] = exp2_4((v[q] - shift) * scale2);
      s += sum4(v[q]);
    }
  } else {
    if (GRAD && !g.row_loss) {
      // The backward has them from the forward: relative to the float next to
      // their log-sum-exp. A rest of up to 16 is off by 2^-21; rows with more
      // below the listed classes (or NaN) are read again.
      const float off = g.rest[row];
      const double at = (double)g.lse[row] + (double)off;
      const float top = (float)(at * g.t);
      known = fabsf(off) <= 16.f && fabsf(top) < -NEG_INF;
      if (known) {
        mr = top;
        s = t == 0 ? (float)exp64(at - (double)top / g.t) : 0.f;
      }
    }
    for (int c0 = known ? c4 : t; c0 < c4; c0 += STREAM_U * RT) {
      f4 r[STREAM_U];
#pragma unroll
      for (int u = 0; u < STREAM_U; ++u) r[u] = *x4(min(c0 + u * RT, c4 - 1));  // plain: the row is read again
      float cm = NEG_INF;
#pragma unroll
      for (int u = 0; u < STREAM_U; ++u) {
        const int c = c0 + u * RT;
        r[u] = without(r[u], c < c4 ? listed(c) : 15u);
        cm = fmaxf(cm, max4(r[u]));
      }
      if (cm > mr) {
        s *= __builtin_amdgcn_exp2f((mr - cm) * scale2);
        mr = cm;
      }
      const float ms = mr == NEG_INF ? 0.f : mr;
#pragma unroll
      for (int u = 0; u < STREAM_U; ++u) s += sum4(exp2_4((r[u] - ms) * scale2));
    }
    const float own = mr;
    maxima();
    s *= own == NEG_INF ? 1.f : __builtin_amdgcn_exp2f((own - mr) * scale2);
  }
  const float shift = shift_of(mr);
  v1 = __builtin_amdgcn_exp2f((v1 - shift) * scale2);
  if (!known) s += v1;
  float total, mine = 0.f, above = 0.f;  // the row's mass; the listed classes' and the others' parts of it
  if constexpr (TAIL) {
#pragma unroll 1
    for (int j = t; j < g.k; j += RT)
      if (eid[j] >= 0) mine += __builtin_amdgcn_exp2f((ex[j] - m) * scale2);
    const Two both = over_block<RT, Both<AddF32>>(Two{s, mine}, reinterpret_cast<Two*>(lds + 2 * (RT / 64)));
    s = both.a;
    mine = both.b;
    above = s * __builtin_amdgcn_exp2f((mr - m) * scale2);
    total = above + mine;
  } else {
    total = s = over_block<RT, AddF32>(s, lds + 2 * (RT / 64));
  }
  if constexpr (GRAD) {
    float* const dr = g.dx + row * C;
    auto put = [&](const f4& d, int c) {
      f4u* const p = reinterpret_cast<f4u*>(reinterpret_cast<char*>(dr + head) + (uint32_t)c * 16u);
      if constexpr (NTS) __builtin_nontemporal_store(d, p);
      else *p = d;
    };
    const float gscale = g.grad_scale(over, up);
    if (some) {
      float gs = gscale / s;
      if constexpr (TAIL)  // s is 1 or more where any of its classes has a finite logit
        gs = s > 0.f || s != s ? gs * rest_excess(psumf, mine / total, above / total, prf, tlse) : 0.f;
      if constexpr (NV > 0) {
#pragma unroll
        for (int q = 0; q < NV; ++q)
          if (q * RT + t < c4) put(v[q] * gs, q * RT + t);
      } else {
        for (int c0 = t; c0 < c4; c0 += STREAM_U * RT) {
          f4 r[STREAM_U];
#pragma unroll
          for (int u = 0; u < STREAM_U; ++u) r[u] = ld_stream(x4(min(c0 + u * RT, c4 - 1)));
#pragma unroll
          for (int u = 0; u < STREAM_U; ++u)
            if (c0 + u * RT < c4) put(exp2_4((r[u] - shift) * scale2) * gs, c0 + u * RT);
        }
      }
      if (has1) dr[e1] = v1 * gs;
    } else {
      for (int c = t; c < c4; c += RT) put(f4{0.f, 0.f, 0.f, 0.f}, c);
      if (has1) dr[e1] = 0.f;
    }
    __syncthreads();  // the entries' own values go over what the row's threads wrote
#pragma unroll 1
    for (int j = t; j < g.k; j += RT) {
      const int id = eid[j];
      if (id < 0) continue;
      double p = ep[j];
      if (twice)
        for (int i = j + 1; i < g.k; ++i)
          if (eid[i] == -2 - id) p += ep[i];
      const float eq = __builtin_amdgcn_exp2f((ex[j] - m) * scale2);
      dr[id] = (float)((double)eq / (double)total - p) * gscale;
    }
    if (!g.row_loss) return;
  }
  const double lt = log64((double)total);
  double terms = 0.0;
#pragma unroll 1
  for (int j = t; j < g.k; j += RT)
    if (eid[j] != -1) terms += entry_term(ep[j], elp[j], ((double)ex[j] - (double)m) / g.t - lt, TAIL, eid[j] <= -2);
  terms = block_sum<RT>(terms, red);
  if (t == 0) {
    double lr = 0.0;
    if constexpr (TAIL) {
      lr = log64((double)s) + ((double)mr - (double)m) / g.t - lt;
      if (some) terms += rest_term(psum_at, lr, tlse);
    }
    write_row(g, row, some, terms, (double)m / g.t + lt, lr);
  }
}

// held[row] = 1 where the row holds an entry, else 0: a wave a row. With the launch
// that adds them up 5 us for 64 entries a row of 8192, 10 for 200 of 16384.
__global__ __launch_bounds__(NT) void distill_held_k(const int64_t* __restrict__ ids, const float* __restrict__ top,
                                                     float* __restrict__ held, int64_t n, int c, int k) {
  const int64_t row = (int64_t)blockIdx.x * (NT / 64) + (threadIdx.x >> 6);
  if (row >= n) return;
  bool any = false;
  for (int j = threadIdx.x & 63; j < k; j += 64) {
    const int64_t id = ids[row * k + j];
    any |= id >= 0 && id < c && top[row * k + j] != NEG_INF;
  }
  const bool some = __ballot(any) != 0;
  if ((threadIdx.x & 63) == 0) held[row] = some ? 1.f : 0.f;
}

// loss[0] = sum of the rows' losses / divisor (count[0], if given), in float64 in a
// fixed order: one block, one round of loads for up to 8192 rows, 4.5 us. Also the
// count of the rows that hold an entry, `least` 1.
__global__ __launch_bounds__(1024) void distill_mean_k(const float* __restrict__ row_loss, int64_t n, double divisor,
                                                       const float* __restrict__ count, float least,
                                                       float* __restrict__ loss) {
  __shared__ double red[1024 / 64];
  constexpr int U = 8;  // loads in flight a thread
  double acc = 0.0;
  for (int64_t i0 = threadIdx.x; i0 < n; i0 += U * 1024) {
    float v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = row_loss[min(i0 + u * 1024, n - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * 1024 < n) acc += (double)v[u];
  }
  acc = block_sum<1024>(acc, red);
  if (threadIdx.x == 0) {
    const float v = (float)(acc / (count ? (double)count[0] : divisor));
    loss[0] = v < least ? least : v;  // a NaN stays
  }
}

int check_distill(const char* what, int64_t n, int64_t c, int64_t k, float temperature, float divisor) {
  if (n < 0 || c < 0 || k < 0) return fail(OXI_INVALID_ARGUMENT, "%s: negative size", what);
  if (c > ((int64_t)1 << 30) || !grid_fits(n, 1024))
    return fail(OXI_INVALID_ARGUMENT, "%s: size exceeds the kernel limits", what);
  if (k < 1 || k > OXI_DISTILL_MAX_TOP)
    return fail(OXI_INVALID_ARGUMENT, "%s: %lld teacher entries a row: 1 to %d are taken", what, (long long)k,
                OXI_DISTILL_MAX_TOP);
  if (!(temperature > 0.f) || std::isinf(temperature))
    return fail(OXI_INVALID_ARGUMENT, "%s: the temperature must be positive, got %g", what, (double)temperature);
  if (std::isinf((float)(1.4426950408889634 / temperature)))  // the kernels' factor of the logits
    return fail(OXI_INVALID_ARGUMENT, "%s: a temperature of %g has no 32-bit reciprocal", what, (double)temperature);
  if (!(divisor > 0.f) || std::isinf(divisor))
    return fail(OXI_INVALID_ARGUMENT, "%s: the divisor must be positive, got %g", what, (double)divisor);
  if (n && c == 0) return fail(OXI_INVALID_ARGUMENT, "%s: zero classes", what);
  return OXI_OK;
}

// The row kernel for c classes and k entries: as few threads as hold the row,
// streamed past 16 float4s on 1024 of them; false where none takes it. A wave alone
// passes no barriers, but works its entries off 64 at a time: 16384 rows of 512
// classes with 256 and 500 entries take 46 and 94 us on it, 65 and 88 on 256
// threads; 8192 rows of 2048 with 64 and 150 31 and 43, 33 and 36.
template <bool GRAD, bool TAIL, bool NTS>
bool launch_rows(const DistillArgs& g) {
  const int c4 = g.c / 4;  // at most
  if (g.c < 8 || g.c > STREAM_MAX) return false;
  const bool one_wave = g.c + 12 * g.k <= 3700;
  const dim3 grid((unsigned)g.n);
  const size_t lds = (size_t)g.k * (2 * sizeof(double) + sizeof(int) + sizeof(float)) + sizeof(uint32_t) * (size_t)bitmap_words(g.c);
  const float scale2 = (float)(1.4426950408889634 / g.t);
#define OXI_DR(RT, NV)                                                                        \
  if ((NV == 0 || c4 <= RT * NV) && (RT > 64 || one_wave)) {                                  \
    distill_rows_k<RT, NV, GRAD, TAIL, NTS><<<grid, dim3(RT), lds, stream()>>>(g, scale2);    \
    return true;                                                                              \
  }
  OXI_DR(64, 2)
  OXI_DR(64, 4)
  OXI_DR(64, 8)
  OXI_DR(64, 16)
  OXI_DR(256, 2)
  OXI_DR(256, 4)
  OXI_DR(256, 6)
  OXI_DR(256, 8)
  OXI_DR(256, 12)
  OXI_DR(256, 16)
  OXI_DR(512, 10)
  OXI_DR(512, 12)
  OXI_DR(512, 14)
  OXI_DR(512, 16)
  OXI_DR(1024, 10)
  OXI_DR(1024, 12)
  OXI_DR(1024, 13)
  OXI_DR(1024, 14)
  OXI_DR(1024, 16)
  OXI_DR(1024, 0)
#undef OXI_DR
  return false;
}

template <bool NTS>
bool launch_rows_any(const DistillArgs& g) {
  if (g.dx) return g.top_lse ? launch_rows<true, true, NTS>(g) : launch_rows<true, false, NTS>(g);
  return g.top_lse ? launch_rows<false, true, false>(g) : launch_rows<false, false, false>(g);
}

void launch_any(const DistillArgs& g) {
  const bool nt = nt_stream_stores(g.n * g.c * 4);
  if (!(nt ? launch_rows_any<true>(g) : launch_rows_any<false>(g)))
    distill_loop_k<<<dim3((unsigned)g.n), dim3(NT), teacher_bytes(g.k), stream()>>>(g);
}

// count: where the divisor lies (formed first), NULL for the one given.
int distill_fwd(const char* what, const float* logits, const int64_t* ids, const float* top, const float* top_lse,
                float* loss, float* row_loss, float* lse, float* rest, float* dlogits, float* count, int64_t n,
                int64_t c, int64_t k, float temperature, float divisor) {
  if (int rc = check_distill(what, n, c, k, temperature, divisor)) return rc;
  if (!loss) return fail(OXI_INVALID_ARGUMENT, "%s: loss must not be NULL", what);
  if (n && (!logits || !ids || !top || !row_loss || !lse || !rest))
    return fail(OXI_INVALID_ARGUMENT, "%s: NULL tensor pointer", what);
  OXI_CHECK_INIT();
  if (n == 0) {
    if (count)
      if (int rc = oxi_fill(count, 1, 1.f)) return rc;
    return oxi_fill(loss, 1, 0.f);
  }
  if (count) {  // the rows' flags lie in row_loss meanwhile
    distill_held_k<<<dim3((unsigned)ceil_div(n, NT / 64)), dim3(NT), 0, stream()>>>(ids, top, row_loss, n, (int)c,
                                                                                     (int)k);
    if (int rc = check_launch(what)) return rc;
    distill_mean_k<<<1, 1024, 0, stream()>>>(row_loss, n, 1.0, nullptr, 1.f, count);
    if (int rc = check_launch(what)) return rc;
  }
  const DistillArgs g{logits, ids,     top, top_lse, row_loss, lse, rest, dlogits, n, (int)c, (int)k,
                      1.0f / temperature, (double)temperature, divisor, count, nullptr, guard_flag()};
  launch_any(g);
  if (int rc = check_launch(what)) return rc;
  distill_mean_k<<<1, 1024, 0, stream()>>>(row_loss, n, (double)divisor, count, -__builtin_huge_valf(), loss);
  return check_launch(what);
}

int distill_bwd(const char* what, const float* logits, const int64_t* ids, const float* top, const float* top_lse,
                const float* lse, const float* rest, const float* gloss, float* dlogits, const float* count, int64_t n,
                int64_t c, int64_t k, float temperature, float divisor) {
  if (int rc = check_distill(what, n, c, k, temperature, divisor)) return rc;
  if (n == 0) return OXI_OK;
  if (!logits || !ids || !top || !lse || !rest || !gloss || !dlogits)
    return fail(OXI_INVALID_ARGUMENT, "%s: NULL tensor pointer", what);
  OXI_CHECK_INIT();
  const DistillArgs g{logits, ids, top, top_lse, nullptr, const_cast<float*>(lse), const_cast<float*>(rest), dlogits, n,
                      (int)c, (int)k, 1.0f / temperature, (double)temperature, divisor, count, gloss, guard_flag()};
  launch_any(g);
  return check_launch(what);
}

}  // namespace
}  // namespace oxi

using namespace oxi;

extern "C" {

int oxi_distill_fwd(const float* logits, const int64_t* ids, const float* top, const float* top_lse, float* loss,
                    float* row_loss, float* lse, float* rest, float* dlogits, int64_t n, int64_t c, int64_t k,
                    float temperature, float divisor) {
  return distill_fwd("distill_fwd", logits, ids, top, top_lse, loss, row_loss, lse, rest, dlogits, nullptr, n, c, k,
                     temperature, divisor);
}

int oxi_distill_fwd_counted(const float* logits, const int64_t* ids, const float* top, const float* top_lse,
                            float* loss, float* row_loss, float* lse, float* rest, float* dlogits, float* count,
                            int64_t n, int64_t c, int64_t k, float temperature) {
  if (!count) return fail(OXI_INVALID_ARGUMENT, "distill_fwd_counted: count must not be NULL");
  return distill_fwd("distill_fwd_counted", logits, ids, top, top_lse, loss, row_loss, lse, rest, dlogits, count, n, c,
                     k, temperature, 1.f);
}

int oxi_distill_bwd(const float* logits, const int64_t* ids, const float* top, const float* top_lse,
                    const float* lse, const float* rest, const float* gloss, float* dlogits, int64_t n, int64_t c,
                    int64_t k, float temperature, float divisor) {
  return distill_bwd("distill_bwd", logits, ids, top, top_lse, lse, rest, gloss, dlogits, nullptr, n, c, k, temperature,
                     divisor);
}

int oxi_distill_bwd_counted(const float* logits, const int64_t* ids, const float* top, const float* top_lse,
                            const float* lse, const float* rest, const float* gloss, float* dlogits,
                            const float* count, int64_t n, int64_t c, int64_t k, float temperature) {
  if (!count) return fail(OXI_INVALID_ARGUMENT, "distill_bwd_counted: count must not be NULL");
  return distill_bwd("distill_bwd_counted", logits, ids, top, top_lse, lse, rest, gloss, dlogits, count, n, c, k,
                     temperature, 1.f);
}

}  // extern "C"

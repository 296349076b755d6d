// Distillation from a teacher's top logits for gfx950: the divergence of a
// student's softmax over c classes from a teacher known by its k best entries a
// row, with its gradient.
//
//   z = x/T, q = exp(z - lse), p the teacher's entries (softmaxed over the row's
//   k, or given the teacher's log-sum-exp, with pr = 1 - sum p left over)
//   row = sum p (log p - log q[id]) + pr (log pr - log qr)
//   dx  = T/divisor (q - p) at the entries, T/divisor q (1 - pr/qr) elsewhere
//
// The k entries of a row are worked out in 64 bits by the block that owns the
// row: a student near its teacher has a small loss of terms that cancel. With
// the rest's term both sides' masses are 1, and the row is summed as
// q - p + p log(p/q), each of which is >= 0, so that an error of lse enters
// squared. qr is the sum over the classes that are not listed, never 1 minus
// the listed.
#include <cmath>

#include "internal.h"
#include "launch_limits.h"
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
  float gscale;  // T / divisor
  int* guard;
};

// A row's teacher entries in LDS: class ids (-1: padding, or an id that an
// earlier entry has, then in `dup`), probabilities and their logarithms.
struct Teacher {
  double* p;
  double* lp;
  int* id;
  int* dup;
};
constexpr size_t teacher_bytes(int64_t k) { return (size_t)k * (2 * sizeof(double) + 2 * sizeof(int)); }

__device__ __forceinline__ Teacher teacher_at(double* lds, int k) {
  Teacher a;
  a.p = lds;
  a.lp = lds + k;
  a.id = reinterpret_cast<int*>(lds + 2 * k);
  a.dup = a.id + k;
  return a;
}

// Sum of doubles over the block, the same bits for every thread; `lds` holds a
// value a wave and is free again after the call.
template <int N>
__device__ __forceinline__ double block_sum(double v, double* lds) {
  v = wave_sum<double>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = lds[0];
#pragma unroll
  for (int i = 1; i < N / 64; ++i) s += lds[i];
  return s;
}

// Fills `a` with the row's entries; returns the sum of p, and whether there is
// any entry in `some`. All threads of the block; the entries are published.
template <int N>
__device__ __forceinline__ double load_teacher(const DistillArgs& g, int64_t row, const Teacher& a, double* red,
                                               bool& some) {
  const int64_t* ids = g.ids + row * g.k;
  const float* top = g.top + row * g.k;
  float* redf = reinterpret_cast<float*>(red);
  float tm = NEG_INF;
  int any = 0;
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
  double s = 0.0;
  for (int j = threadIdx.x; j < g.k; j += N) {
    const bool there = a.id[j] >= 0;
    const double v = a.lp[j];
    const double l = g.top_lse ? v / g.t - (double)g.top_lse[row] : (v - (double)tm) / g.t;
    const double p = there ? exp(l) : 0.0;
    a.lp[j] = l;
    a.p[j] = p;
    s += p;
    int d = -1;
    if (there)
      for (int i = 0; i < j && d < 0; ++i)
        if (a.id[i] == a.id[j]) d = i;
    a.dup[j] = d;
  }
  s = block_sum<N>(s, red);
  if (!g.top_lse && some) {  // divide by the sum
    const double ls = log(s);
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
  return p > 0.0 || p != p ? p * (expm1(d) - d) : exp(lq);
}

// The loss of the row once its maximum, its sum of exp((x - m)/T) and, with
// the rest's term, the sum over the classes not listed are known; thread 0 writes
// the row's results. Returns the factor of q at the classes not listed.
template <int N>
__device__ __forceinline__ float finish_row(const DistillArgs& g, int64_t row, const Teacher& a, double* red,
                                            double psum, bool some, float m, double total, double rest) {
  const bool tail = g.top_lse != nullptr;
  const double lt = log(total);
  const float* xr = g.x + row * g.c;
  double s = 0.0;
  for (int j = threadIdx.x; j < g.k; j += N)
    if (a.id[j] >= 0)
      s += entry_term(a.p[j], a.lp[j], ((double)xr[a.id[j]] - (double)m) / g.t - lt, tail, a.dup[j] >= 0);
  s = block_sum<N>(s, red);
  float factor = 1.f;
  const double lr = tail ? log(rest) - lt : 0.0;
  if (tail && some) {
    const double pr = psum < 1.0 ? 1.0 - psum : psum != psum ? psum : 0.0;
    const double qr = rest / total;
    const double d = lr - log(pr);
    s += pr > 0.0 || pr != pr ? pr * (expm1(d) - d) : qr;
    s += (psum + pr) - 1.0;
    factor = qr > 0.0 || qr != qr ? (float)((qr - pr) / qr) : 1.f;
  }
  if (threadIdx.x == 0) {
    g.row_loss[row] = some ? (float)(g.t * g.t * s) : 0.f;
    g.lse[row] = (float)((double)m / g.t + lt);
    g.rest[row] = tail ? (float)lr : 0.f;
  }
  return some ? factor : 0.f;
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
    double p = 0.0;
    for (int i = j; i < g.k; ++i)
      if (a.id[i] == id) p += a.p[i];
    dr[id] = (float)(q(id) - p) * gscale;
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

// A block a row of any length, which it walks three times.
__global__ __launch_bounds__(NT) void distill_fwd_k(const DistillArgs g) {
  extern __shared__ __align__(16) double dyn[];
  __shared__ double red[NT / 64];
  __shared__ uint32_t bits[STRETCH / 32];
  const Teacher a = teacher_at(dyn, g.k);
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  const float* xr = g.x + row * g.c;
  bool some;
  const double psum = load_teacher<NT>(g, row, a, red, some);
  float m = NEG_INF;
  for (int c = t; c < g.c; c += NT) m = fmaxf(m, xr[c]);
  m = group_max<NT>(m, reinterpret_cast<float*>(red));
  double total = 0.0, listed = 0.0, rest = 0.0;
  if (g.top_lse) {
    for (int c0 = 0; c0 < g.c; c0 += STRETCH) {
      mark_listed<NT>(a, g.k, c0, bits);
      const int end = min(g.c - c0, STRETCH);
      for (int c = t; c < end; c += NT) {
        const double e = expf((xr[c0 + c] - m) * g.inv_t);
        if (bits[c >> 5] >> (c & 31) & 1) listed += e;
        else rest += e;
      }
    }
    rest = block_sum<NT>(rest, red);
    total = rest + block_sum<NT>(listed, red);
  } else {
    for (int c = t; c < g.c; c += NT) total += expf((xr[c] - m) * g.inv_t);
    total = block_sum<NT>(total, red);
  }
  const float factor = finish_row<NT>(g, row, a, red, psum, some, m, total, rest);
  if (!g.dx) return;
  const float scale = (float)(1.0 / total) * g.gscale;
  float* dr = g.dx + row * g.c;
  for (int c = t; c < g.c; c += NT) {
    const float e = expf((xr[c] - m) * g.inv_t) * scale;
    dr[c] = some ? e * factor : 0.f;
  }
  write_entries<NT>(g, row, a, g.gscale,
                    [&](int id) { return (double)expf((xr[id] - m) * g.inv_t) / total; });
}

// ---------------------------------------------------------------------------
// Rows of up to RT * NV float4s at any float alignment, a row per block held in
// registers, so the logits cross HBM once for the loss and its gradient. The row
// group waits for its logits first, and works out the teacher's entries
// meanwhile. Exponentials are exp2 of (x - m) * (log2(e)/T).

// What an entry needs later, kept by its thread: k <= RT entries, thread j's
// at j.
struct Entry {
  double p, lp;
  float x;   // the student's logit
  int id;    // -1: padding
  bool dup;  // an earlier entry has this id
};

// Bits of slot c's four classes (bit j: class first + j is listed).
template <int KIND>
__device__ __forceinline__ uint32_t listed_bits(const uint32_t* bits, int C, int c) {
  if constexpr (KIND == ROW_ODD) {
    const int e = min(4 * c, C - 4);
    const uint64_t two = (uint64_t)bits[e >> 5] | (uint64_t)bits[(e >> 5) + 1] << 32;
    return (uint32_t)(two >> (e & 31)) & 15u;
  } else {
    return bits[c >> 3] >> ((c & 7) * 4) & 15u;
  }
}

// NV = 0: longer rows, streamed twice, the first time with a running maximum; the
// second time they come from the Infinity Cache (a block a row on every CU is
// at most 256 rows in flight, 134 MB of 131072 classes).
constexpr int STREAM_U = 4;         // float4s in flight a thread
constexpr int STREAM_MAX = 400000;  // classes whose bitmap fits in LDS beside 1024 entries

__device__ __forceinline__ f4 exp2_4(const f4& z) {
  return f4{__builtin_amdgcn_exp2f(z.x), __builtin_amdgcn_exp2f(z.y), __builtin_amdgcn_exp2f(z.z),
            __builtin_amdgcn_exp2f(z.w)};
}

template <int RT, int NV, int KIND, bool GRAD, bool TAIL, bool NTS>
__global__ __launch_bounds__(RT) void distill_rows_k(const DistillArgs g, const float scale2) {
  __shared__ double red[RT / 64];
  __shared__ float lds[2 * (RT / 64)];
  __shared__ int twice;
  extern __shared__ __align__(16) double dyn[];  // k probabilities, k ids, a bit a class
  double* const ep = dyn;
  int* const eid = reinterpret_cast<int*>(dyn + g.k);
  uint32_t* const bits = reinterpret_cast<uint32_t*>(eid + g.k);
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int C = g.c;
  const int h4 = row_slots<KIND>(C);
  const float* xr = g.x + row * C;
  // the entries' loads go first: a wait for them leaves the row's in flight
  const int64_t id64 = t < g.k ? g.ids[row * g.k + t] : -1;
  const float top = t < g.k ? g.top[row * g.k + t] : 0.f;
  const float tlse = TAIL ? g.top_lse[row] : 0.f;
  // the plain load keeps a row that is read again in the caches
  auto load = [&](int c) -> f4 {
    if constexpr (KIND == ROW_ODD) return ld_odd(xr, C, c);
    else if constexpr (NV == 0) return reinterpret_cast<const f4*>(xr)[min(c, h4 - 1)];
    else return ld_stream(reinterpret_cast<const f4*>(xr) + min(c, h4 - 1));
  };
  f4 v[NV ? NV : 1];
#pragma unroll
  for (int q = 0; q < NV; ++q) v[q] = load(q * RT + t);
  for (int i = t; i < (C >> 5) + 2; i += RT) bits[i] = 0;
  if (t == 0) twice = 0;
  Entry e;
  e.id = t < g.k && id64 >= 0 && id64 < C && top != NEG_INF ? (int)id64 : -1;
  e.dup = false;
  e.x = e.id >= 0 ? xr[e.id] : 0.f;
  if (t < g.k && id64 >= C) atomicOr(g.guard, 1);
  const bool there = e.id >= 0;
  if (t < g.k) eid[t] = e.id;
  const bool some = __syncthreads_or(there) != 0;  // and the bitmap is clear
  if (there) {
    const uint32_t bit = 1u << (e.id & 31);
    if (atomicOr(bits + (e.id >> 5), bit) & bit) twice = 1;
  }
  double psum;
  if constexpr (TAIL) {
    e.lp = there ? (double)top / g.t - (double)tlse : 0.0;
    e.p = there ? exp(e.lp) : 0.0;
    psum = block_sum<RT>(e.p, red);  // its barriers publish the bitmap
  } else {
    const float tm = group_max<RT>(there ? top : NEG_INF, lds);
    e.lp = there ? ((double)top - (double)tm) / g.t : 0.0;
    e.p = there ? exp(e.lp) : 0.0;
    psum = block_sum<RT>(e.p, red);
    e.p = there ? e.p / psum : 0.0;
    e.lp -= log(psum);
  }
  if (t < g.k) ep[t] = e.p;
  if (twice) {  // ids given twice: rare, so their order is looked up only then
    if (there)
      for (int i = 0; i < t && !e.dup; ++i) e.dup = eid[i] == e.id;
  }
  // the unlisted (TAIL) or all of slot c's exponentials
  auto counted = [&](const f4& ev, int c) -> float {
    f4 u = without_dup<KIND>(ev, C, c);
    if constexpr (TAIL) {
      const uint32_t b = listed_bits<KIND>(bits, C, c);
      u.x = b & 1 ? 0.f : u.x;
      u.y = b & 2 ? 0.f : u.y;
      u.z = b & 4 ? 0.f : u.z;
      u.w = b & 8 ? 0.f : u.w;
    }
    return sum4(u);
  };
  float m = NEG_INF, s = 0.f;
  if constexpr (NV > 0) {
#pragma unroll
    for (int q = 0; q < NV; ++q) m = fmaxf(m, max4(v[q]));  // slots past the row repeat its last
    m = group_max<RT>(m, lds);
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      v[q] = exp2_4((v[q] - m) * scale2);
      if (q * RT + t < h4) s += counted(v[q], q * RT + t);
    }
  } else {
    for (int c0 = t; c0 < h4; c0 += STREAM_U * RT) {
      f4 r[STREAM_U];
#pragma unroll
      for (int u = 0; u < STREAM_U; ++u) r[u] = load(c0 + u * RT);
      float cm = max4(r[0]);
#pragma unroll
      for (int u = 1; u < STREAM_U; ++u) cm = fmaxf(cm, max4(r[u]));
      if (cm > m) {
        s *= __builtin_amdgcn_exp2f((m - cm) * scale2);
        m = cm;
      }
      const float ms = m == NEG_INF ? 0.f : m;
#pragma unroll
      for (int u = 0; u < STREAM_U; ++u)
        if (c0 + u * RT < h4) s += counted(exp2_4((r[u] - ms) * scale2), c0 + u * RT);
    }
    const float own = m;
    m = group_max<RT>(m, lds);
    s *= own == NEG_INF ? 0.f : __builtin_amdgcn_exp2f((own - m) * scale2);
  }
  double total = (double)group_sum<RT, float>(s, lds + RT / 64);
  const double rest = total;
  const float ex = there ? __builtin_amdgcn_exp2f((e.x - m) * scale2) : 0.f;
  if constexpr (TAIL) total += block_sum<RT>(e.dup ? 0.0 : (double)ex, red);
  const double pr = psum < 1.0 ? 1.0 - psum : psum != psum ? psum : 0.0;
  if constexpr (GRAD) {
    float factor = some ? 1.f : 0.f;
    if constexpr (TAIL)
      if (some) {
        const double qr = rest / total;
        factor = qr > 0.0 || qr != qr ? (float)((qr - pr) / qr) : 1.f;
      }
    const float gs = some ? (float)(1.0 / total) * g.gscale * factor : 0.f;
    float* dr = g.dx + row * C;
    auto put = [&](const f4& ev, int c) {
      const f4 d = some ? ev * gs : f4{0.f, 0.f, 0.f, 0.f};
      if constexpr (KIND == ROW_ODD) *reinterpret_cast<f4u*>(dr + min(4 * c, C - 4)) = d;
      else st_stream<NTS>(d, reinterpret_cast<f4*>(dr) + c);
    };
    if constexpr (NV > 0) {
#pragma unroll
      for (int q = 0; q < NV; ++q)
        if (q * RT + t < h4) put(v[q], q * RT + t);
    } else {
      for (int c0 = t; c0 < h4; c0 += STREAM_U * RT) {
        f4 r[STREAM_U];
#pragma unroll
        for (int u = 0; u < STREAM_U; ++u) r[u] = load(c0 + u * RT);
#pragma unroll
        for (int u = 0; u < STREAM_U; ++u)
          if (c0 + u * RT < h4) put(exp2_4((r[u] - m) * scale2), c0 + u * RT);
      }
    }
    __syncthreads();  // the entries' own values go over what the row's threads wrote
    if (there && !e.dup) {
      double p = e.p;
      if (twice)
        for (int i = t + 1; i < g.k; ++i)
          if (eid[i] == e.id) p += ep[i];
      dr[e.id] = (float)((double)ex / total - p) * g.gscale;
    }
  }
  const double lt = log(total);
  double terms = there ? entry_term(e.p, e.lp, ((double)e.x - (double)m) / g.t - lt, TAIL, e.dup) : 0.0;
  terms = block_sum<RT>(terms, red);
  if (t == 0) {
    double lr = 0.0;
    if constexpr (TAIL) {
      lr = log(rest) - lt;
      if (some) {
        const double d = lr - log(pr);
        terms += pr > 0.0 || pr != pr ? pr * (expm1(d) - d) : rest / total;
        terms += (psum + pr) - 1.0;
      }
    }
    g.row_loss[row] = some ? (float)(g.t * g.t * terms) : 0.f;
    g.lse[row] = (float)((double)m / g.t + lt);
    g.rest[row] = (float)lr;
  }
}

// The gradient from the forward's log-sum-exp and rest, for an upstream scalar.
__global__ __launch_bounds__(NT) void distill_bwd_k(const DistillArgs g, const float* __restrict__ gloss) {
  extern __shared__ __align__(16) double dyn[];
  __shared__ double red[NT / 64];
  const Teacher a = teacher_at(dyn, g.k);
  const int64_t row = blockIdx.x;
  const float* xr = g.x + row * g.c;
  bool some;
  const double psum = load_teacher<NT>(g, row, a, red, some);
  const float scale = g.gscale * gloss[0];
  const float l = g.lse[row];
  float factor = 1.f;
  if (g.top_lse && some) {
    const double pr = psum < 1.0 ? 1.0 - psum : psum != psum ? psum : 0.0;
    const double qr = exp((double)g.rest[row]);
    factor = qr > 0.0 || qr != qr ? (float)((qr - pr) / qr) : 1.f;
  }
  float* dr = g.dx + row * g.c;
  for (int c = threadIdx.x; c < g.c; c += NT) {
    const float e = expf(xr[c] * g.inv_t - l) * scale;
    dr[c] = some ? e * factor : 0.f;
  }
  write_entries<NT>(g, row, a, scale, [&](int id) { return (double)expf(xr[id] * g.inv_t - l); });
}

// loss[0] = sum of the rows' losses / divisor, in float64 in a fixed order.
__global__ __launch_bounds__(1024) void distill_mean_k(const float* __restrict__ row_loss, int64_t n, double divisor,
                                                       float* __restrict__ loss) {
  __shared__ double red[1024 / 64];
  double acc = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) acc += (double)row_loss[i];
  acc = block_sum<1024>(acc, red);
  if (threadIdx.x == 0) loss[0] = (float)(acc / divisor);
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
  if (!(divisor > 0.f) || std::isinf(divisor))
    return fail(OXI_INVALID_ARGUMENT, "%s: the divisor must be positive, got %g", what, (double)divisor);
  if (n && c == 0) return fail(OXI_INVALID_ARGUMENT, "%s: zero classes", what);
  return OXI_OK;
}

// The register kernel for rows of c floats with k entries: 16 float4s a thread, 8
// for rows of 16385 to 32768 floats, longer rows streamed; false when none takes them.
template <int KIND, bool GRAD, bool TAIL, bool NTS>
bool launch_rows(const DistillArgs& g) {
  const int h4 = (g.c + 3) / 4;
  const dim3 grid((unsigned)g.n);
  const size_t lds = (size_t)g.k * (sizeof(double) + sizeof(int)) + sizeof(uint32_t) * ((size_t)(g.c >> 5) + 2);
  const float scale2 = (float)(1.4426950408889634 / g.t);
#define OXI_DR(RT, NV)                                                                              \
  if (h4 <= RT * NV && g.k <= RT) {                                                                 \
    distill_rows_k<RT, NV, KIND, GRAD, TAIL, NTS><<<grid, dim3(RT), lds, stream()>>>(g, scale2);    \
    return true;                                                                                    \
  }
  OXI_DR(64, 4)
  OXI_DR(64, 16)
  OXI_DR(128, 16)
  OXI_DR(256, 16)
  OXI_DR(1024, 8)
  OXI_DR(1024, 16)
#undef OXI_DR
  if (g.c > STREAM_MAX) return false;
  distill_rows_k<1024, 0, KIND, GRAD, TAIL, NTS><<<grid, dim3(1024), lds, stream()>>>(g, scale2);
  return true;
}

template <int KIND, bool NTS>
bool launch_rows_kind(const DistillArgs& g) {
  if (g.dx) return g.top_lse ? launch_rows<KIND, true, true, NTS>(g) : launch_rows<KIND, true, false, NTS>(g);
  return g.top_lse ? launch_rows<KIND, false, true, false>(g) : launch_rows<KIND, false, false, false>(g);
}

bool launch_rows_any(const DistillArgs& g) {
  if (g.c < 4) return false;
  const bool odd = g.c % 4 || (reinterpret_cast<uintptr_t>(g.x) & 15u) || (reinterpret_cast<uintptr_t>(g.dx) & 15u);
  if (odd) return launch_rows_kind<ROW_ODD, false>(g);
  return nt_stores(g.n * g.c * 4) ? launch_rows_kind<ROW_VEC, true>(g) : launch_rows_kind<ROW_VEC, false>(g);
}

}  // namespace
}  // namespace oxi

using namespace oxi;

extern "C" {

int oxi_distill_fwd(const float* logits, const int64_t* ids, const float* top, const float* top_lse, float* loss,
                    float* row_loss, float* lse, float* rest, float* dlogits, int64_t n, int64_t c, int64_t k,
                    float temperature, float divisor) {
  if (int rc = check_distill("distill_fwd", n, c, k, temperature, divisor)) return rc;
  if (!loss) return fail(OXI_INVALID_ARGUMENT, "distill_fwd: loss must not be NULL");
  if (n && (!logits || !ids || !top || !row_loss || !lse || !rest))
    return fail(OXI_INVALID_ARGUMENT, "distill_fwd: NULL tensor pointer");
  OXI_CHECK_INIT();
  if (n == 0) return oxi_fill(loss, 1, 0.f);
  const DistillArgs g{logits, ids,    top, top_lse, row_loss,           lse,         rest, dlogits, n, (int)c,
                      (int)k, 1.0f / temperature, (double)temperature, temperature / divisor, guard_flag()};
  if (!launch_rows_any(g)) distill_fwd_k<<<dim3((unsigned)n), dim3(NT), teacher_bytes(k), stream()>>>(g);
  if (int rc = check_launch("distill_fwd")) return rc;
  distill_mean_k<<<1, 1024, 0, stream()>>>(row_loss, n, (double)divisor, loss);
  return check_launch("distill_fwd: mean");
}

int oxi_distill_bwd(const float* logits, const int64_t* ids, const float* top, const float* top_lse,
                    const float* lse, const float* rest, const float* gloss, float* dlogits, int64_t n, int64_t c,
                    int64_t k, float temperature, float divisor) {
  if (int rc = check_distill("distill_bwd", n, c, k, temperature, divisor)) return rc;
  if (n == 0) return OXI_OK;
  if (!logits || !ids || !top || !lse || !rest || !gloss || !dlogits)
    return fail(OXI_INVALID_ARGUMENT, "distill_bwd: NULL tensor pointer");
  OXI_CHECK_INIT();
  const DistillArgs g{logits, ids,    top, top_lse, nullptr, const_cast<float*>(lse), const_cast<float*>(rest), dlogits, n,
                      (int)c, (int)k, 1.0f / temperature, (double)temperature, temperature / divisor, guard_flag()};
  distill_bwd_k<<<dim3((unsigned)n), dim3(NT), teacher_bytes(k), stream()>>>(g, gloss);
  return check_launch("distill_bwd");
}

}  // extern "C"

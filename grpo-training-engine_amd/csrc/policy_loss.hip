// The policy update's loss on gfx950: log-probabilities of given tokens under a
// vocabulary of logits, the clipped policy loss with a KL term, and the gradients of both.
//
// For a counted row of logits x, its token id, T > 0 and k = log2(e) / T:
//   S    = sum_v exp2(x_v k - M)              M: an integer near max(x) k
//   logp = ln 2 (x_id k - M - log2 S)          H = ln 2 (log2 S - sum_v e_v (x_v k - M) / S)
//   d loss / d x_v = c / T (1[v = id] - e_v / S),  c = d loss / d logp
// and for the loss, with r = exp(logp - old) and the advantage A of a token,
//   g = min(min(r, delta) A, clip(r, 1 - lo, 1 + hi) A),  q = ref - logp
//   l = beta (exp(q) - q - 1) - g,  loss = sum w l
//   d l / d logp = (g follows r ? -r A : 0) + beta (1 - exp(q))
// with w = 1 / (counted tokens), 1 / (counted tokens of the row's sequence x counted
// sequences) or 1 / (a given number). Rows that are not counted are not read: their
// logp, loss and gradient are 0 whatever stands there.
//
// x k - M is two fused multiply-adds, k = khi + klo: each rounds at the size of its result,
// whatever offset the logits have in common. (With k rounded to float32 every logp of a
// batch moves the same way, and a loss whose advantages cancel shows it: 1.4e-5 relative at
// T = 0.7, 5e-8 with both.) M is an integer, so sums taken against different M are brought
// together by exact powers of two. Everything per row is float64 from the threads' sums on:
// the ratio of a token next to a border of the clip decides whether it has a gradient at all.
//
// All of it is bound by the logits' way through memory; two exponentials a value keep the
// vector units at about half of that time.
//  * log-probabilities: a workgroup a row, eight 16-byte loads of a thread on their way;
//    few rows are cut over several workgroups and joined. 2994 counted rows of 151936 bf16 in
//    155 us, 5.9 TB/s; 8 rows 8.1 us (17.3 with one workgroup each).
//  * the loss with the logits' gradient: a row stays in the registers of one workgroup
//    (loss_rows_kernel), so the logits are read once and their gradient written once. 4096
//    rows of 151936 bf16, three quarters of them counted, in 406 us: 2.18 GB at 5.4 TB/s (a
//    copy of 1 GiB runs at 4.8 to 5.15), where a pass for the sums and one for the gradient
//    took 168 + 409. A few long rows still take these two.
//  * the loss from log-probabilities: 17 bytes a token; its time is that of its launches.
#include <type_traits>
#include <algorithm>

#include "common.hpp"

using namespace grpo;

namespace {

enum Dtype { BF16 = 0, F16 = 1, F32 = 2 };
constexpr float LOWEST = -1e30f;  // M of what has no finite logit above -1e30
constexpr double LN2 = 0.693147180559945309417;

// A batch of rows of logits: row r = (b, s) = (r / S, r % S) starts at b sb + s ss.
struct Rows {
  const void* x;
  int64_t sb, ss;
  int S, V;
  const int64_t* ids;   // [rows]
  const uint8_t* mask;  // [rows] or null: every row is counted
  double k;             // log2(e) / T
  float khi, klo;       // khi < k, khi + klo = k; klo > 0 keeps -inf * klo from being NaN
};
// (Rows is never passed by reference to a function that is not inlined: it would have to
// live in memory, and its pointers would no longer be known to be global.)

// What the gradient needs of a row: e_v = exp2(x_v k - M), or exp2((x_v - m) khi) where M
// is not finite (rows whose logits are all below -1e30, or not finite). S in float32, as is
// -c / S made of it: a rounding of 2^-24 each, where e_v's exponential alone is off by 2^-23.
struct RowStat {
  float M, S, m, pad;
};

__device__ __forceinline__ float exponent(float x, float khi, float klo, float M) {
  return fmaf(x, klo, fmaf(x, khi, -M));
}

using Policy = grpo_policy_t;

template <int DT>
using Raw = std::conditional_t<DT == F32, float, uint16_t>;
template <int DT>
__device__ __forceinline__ Raw<DT> load_raw(const void* x, int64_t i) {
  return static_cast<const Raw<DT>*>(x)[i];
}
template <int DT>
__device__ __forceinline__ float to_float(Raw<DT> v) {
  if constexpr (DT == F32) return v;
  else return e2f<DT == F16>(v);
}
template <int DT>
__device__ __forceinline__ float load1(const void* x, int64_t i) {
  return to_float<DT>(load_raw<DT>(x, i));
}
template <int DT>
__device__ __forceinline__ void store1(void* x, int64_t i, float v) {
  if (DT == F32) static_cast<float*>(x)[i] = v;
  else static_cast<uint16_t*>(x)[i] = f2e<DT == F16>(v);
}
template <int DT>
constexpr int SIZE = DT == F32 ? 4 : 2;
template <int DT>
constexpr int PER = 16 / SIZE<DT>;  // values of a 16-byte load

template <int DT>
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[PER<DT>]) {
  const uint32_t d[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (DT == F32) {
      f[q] = __uint_as_float(d[q]);
    } else {
      f[2 * q] = e2f<DT == F16>((uint16_t)d[q]);
      f[2 * q + 1] = e2f<DT == F16>((uint16_t)(d[q] >> 16));
    }
  }
}
template <int DT>
__device__ __forceinline__ uint4 pack(const float (&f)[PER<DT>]) {
  uint32_t d[4];
#pragma unroll
  for (int q = 0; q < 4; ++q)
    d[q] = DT == F32 ? __float_as_uint(f[q]) : pack_e2<DT == F16>(f[2 * q], f[2 * q + 1]);
  return make_uint4(d[0], d[1], d[2], d[3]);
}

// Values before the first 16-byte boundary at or after p.
template <int DT>
__device__ __forceinline__ int head_of(const void* p, int n) {
  return min(n, (int)((-reinterpret_cast<uintptr_t>(p) & 15u) / SIZE<DT>));
}

// ------------------------------------------------------- softmax statistics --

// A difference of two Ms as ldexp takes it; beyond 2^-4096 nothing is left anyway.
__device__ __forceinline__ int shift(float d) { return (int)fmaxf(d, -4096.f); }

// S, and t = sum e (x k - M) for the entropy, against an M of its own. What is added is at
// most 2^4: its exponent x k - M is rounded at 4 at most, so the largest terms are exact to
// little more than the exponential's own last bit; the sums are float64, one addition for
// each N terms that were added to each other in float32.
template <bool ENT>
struct Sums {
  float M = LOWEST;
  double S = 0.0, t = 0.0;
  __device__ __forceinline__ void admit(float top, const Rows& q) {
    if (top * q.khi > M + 4.f) {
      const float to = rintf(top * q.khi) + 4.f;
      const int by = shift(M - to);
      if (ENT) t = ldexp(t + (double)(M - to) * S, by);
      S = ldexp(S, by);
      M = to;
    }
  }
  template <int N>
  __device__ __forceinline__ void add(const float (&x)[N], const Rows& q) {
    float e[N], u[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float a = exponent(x[j], q.khi, q.klo, M);
      e[j] = __builtin_amdgcn_exp2f(a);
      u[j] = ENT ? e[j] * fmaxf(a, -1024.f) : 0.f;  // a = -inf: 0, not 0 * inf
    }
#pragma unroll
    for (int w = 1; w < N; w *= 2)
#pragma unroll
      for (int j = 0; j + w < N; j += 2 * w) {
        e[j] += e[j + w];
        if (ENT) u[j] += u[j + w];
      }
    S += e[0];
    if (ENT) t += u[0];
  }
};

// Over the 64 lanes of a wave, every lane gets the result (as wave_sum_dpp).
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp_move<0xB1>(v));
  v = fmaxf(v, dpp_move<0x4E>(v));
  v = fmaxf(v, dpp_move<0x141>(v));
  v = fmaxf(v, dpp_move<0x140>(v));
  return pair32_max(pair16_max(v));
}
template <int CTRL>
__device__ __forceinline__ double dpp_move64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum64(double v) {
  v += dpp_move64<0xB1>(v);
  v += dpp_move64<0x4E>(v);
  v += dpp_move64<0x141>(v);
  v += dpp_move64<0x140>(v);
  uint64_t u = __builtin_bit_cast(uint64_t, v);
  auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)u, (uint32_t)u, false, false);
  auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
  v = __builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]) +
      __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]);
  u = __builtin_bit_cast(uint64_t, v);
  lo = __builtin_amdgcn_permlane32_swap((uint32_t)u, (uint32_t)u, false, false);
  hi = __builtin_amdgcn_permlane32_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
  return __builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]) +
         __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]);
}

struct Joined {  // of a workgroup, the same in every thread
  float M;
  double S, t;
};
template <int NT>
struct JoinSpace {
  double S[NT / 64], t[NT / 64];
  float M[NT / 64];
};

// A wave's sums against the largest M among its lanes.
template <bool ENT>
__device__ __forceinline__ Joined join_wave(float M, double S, double t) {
  const float top = wave_max(M);
  const int by = shift(M - top);
  return Joined{top, wave_sum64(ldexp(S, by)),
                ENT ? wave_sum64(ldexp(t + (double)(M - top) * S, by)) : 0.0};
}
// The waves' sums into LDS ...
template <bool ENT, int NT>
__device__ __forceinline__ void leave(const Sums<ENT>& s, JoinSpace<NT>& red) {
  const Joined w = join_wave<ENT>(s.M, s.S, s.t);
  if ((threadIdx.x & 63) == 0) {
    red.M[threadIdx.x >> 6] = w.M;
    red.S[threadIdx.x >> 6] = w.S;
    if (ENT) red.t[threadIdx.x >> 6] = w.t;
  }
}
// ... and joined by any wave, a lane each, after a barrier.
template <bool ENT, int NT>
__device__ __forceinline__ Joined gather(const JoinSpace<NT>& red) {
  const int l = threadIdx.x & 63;
  const bool in = l < NT / 64;
  return join_wave<ENT>(in ? red.M[l] : LOWEST, in ? red.S[l] : 0.0, in && ENT ? red.t[l] : 0.0);
}
template <bool ENT, int NT>
__device__ __forceinline__ Joined join(const Sums<ENT>& s, JoinSpace<NT>& red) {
  __syncthreads();
  leave<ENT, NT>(s, red);
  __syncthreads();
  return gather<ENT, NT>(red);
}
// Whether S can be the sum of up to 2^30 terms of which the largest is near 1. Beyond: nothing
// above -1e30, values that are not finite, or |x k| so large (2^27) that M, a float32, is no
// longer near it.
__device__ __forceinline__ bool usable(const Joined& j) { return j.S > 0x1p-8 && j.S < 0x1p40; }

template <int NT>
__device__ __forceinline__ double block_sum64(double v, JoinSpace<NT>& red) {
  v = wave_sum64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red.S[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
  for (int w = 0; w < NT / 64; ++w) v += red.S[w];
  return v;
}

// A row as one workgroup sees it: vectors from the first 16-byte boundary on, and the
// fewer than 2 PER values around them, one a thread.
template <int DT>
struct Span {
  const void* row;
  const uint4* vec;
  int head, nvec, tail, odd;
  __device__ __forceinline__ Span(const void* p, int V) : row(p) {
    head = head_of<DT>(p, V);
    nvec = (V - head) / PER<DT>;
    tail = head + nvec * PER<DT>;
    odd = head + V - tail;
    vec = reinterpret_cast<const uint4*>(static_cast<const char*>(p) + (int64_t)head * SIZE<DT>);
  }
  __device__ __forceinline__ int odd_at(int i) const { return i < head ? i : tail + i - head; }
};

template <int DT>
__device__ __forceinline__ float top_of(const float (&f)[PER<DT>]) {
  float top = f[0];
#pragma unroll
  for (int j = 1; j < PER<DT>; ++j) top = fmaxf(top, f[j]);
  return top;
}

// The statistics of a row whose sums are not usable: the maximum, then the sum against it.
struct PlainStat {
  double S, t;
  float m;
};
template <int DT, bool ENT, int NT>
__device__ __noinline__ PlainStat plain_stat(const void* row, int V, float k, float* red) {
  __syncthreads();
  float top = -INFINITY;
  for (int v = threadIdx.x; v < V; v += NT) top = fmaxf(top, load1<DT>(row, v));
  top = wave_max(top);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
  for (int w = 0; w < NT / 64; ++w) top = fmaxf(top, red[w]);
  double S = 0.0, t = 0.0;
  for (int v = threadIdx.x; v < V; v += NT) {
    const float a = (load1<DT>(row, v) - top) * k, e = __builtin_amdgcn_exp2f(a);
    S += e;
    if (ENT) t += e * fmaxf(a, -1024.f);
  }
  double* const sum = reinterpret_cast<double*>(red);
  S = wave_sum64(S);
  t = wave_sum64(t);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    sum[threadIdx.x >> 6] = S;
    sum[NT / 64 + (threadIdx.x >> 6)] = t;
  }
  __syncthreads();
  S = t = 0.0;
  for (int w = 0; w < NT / 64; ++w) {
    S += sum[w];
    t += sum[NT / 64 + w];
  }
  return PlainStat{S, t, top};
}

// Vectors [i0, i1) of a row, and the values around the vectors if `odd`, added to s; AHEAD
// vectors of a thread are on their way.
template <int DT, bool ENT, bool ONCE, int NT, int AHEAD = 8>
__device__ __forceinline__ void add_span(const Span<DT>& sp, int i0, int i1, bool odd,
                                         const Rows& q, Sums<ENT>& s) {
  auto load = [&](int i) __attribute__((always_inline)) {
    return ONCE ? load_stream(sp.vec + i) : sp.vec[i];
  };
  auto take = [&](const uint4& v) __attribute__((always_inline)) {
    float f[PER<DT>];
    unpack<DT>(v, f);
    s.admit(top_of<DT>(f), q);
    s.add(f, q);
  };
  int i = i0 + (int)threadIdx.x;
  for (; i + (AHEAD - 1) * NT < i1; i += AHEAD * NT) {
    uint4 v[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) v[j] = load(i + j * NT);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) take(v[j]);
  }
  for (; i < i1; i += NT) take(load(i));
  if (odd && (int)threadIdx.x < sp.odd) {
    const float x[1] = {load1<DT>(sp.row, sp.odd_at(threadIdx.x))};
    s.admit(x[0], q);
    s.add(x, q);
  }
}

// The statistics of a row from its threads' sums, and what the row's gradient needs of them.
template <int DT, bool ENT, int NT>
__device__ __forceinline__ Joined row_stat(const Sums<ENT>& s, const void* row, const Rows& q,
                                           JoinSpace<NT>& red, RowStat* st) {
  Joined j = join<ENT, NT>(s, red);
  float m = 0.f;
  if (!usable(j)) {
    const PlainStat ps =
        plain_stat<DT, ENT, NT>(row, q.V, q.khi, reinterpret_cast<float*>(&red));
    j = Joined{INFINITY, ps.S, ps.t};
    m = ps.m;
  }
  *st = RowStat{j.M, (float)j.S, m, 0.f};
  return j;
}

// The row's value at its token; NaN for an id outside the vocabulary.
template <int DT>
__device__ __forceinline__ float row_at_id(const void* row, int64_t id, int V) {
  return id < 0 || id >= V ? __builtin_nanf("") : load1<DT>(row, id);
}
// Its exponent: logp is ln 2 (this - log2 S).
__device__ __forceinline__ double id_exponent(float x, const Rows& q, const Joined& j, float m) {
  return j.M < INFINITY ? fma((double)x, q.k, -(double)j.M)
                        : ((double)x - (double)m) * (double)q.khi;
}

template <int DT>
__device__ __forceinline__ const void* row_at(const Rows& q, int64_t r) {
  const uint32_t b = (uint32_t)r / (uint32_t)q.S, s = (uint32_t)r - b * q.S;  // < 2^22 rows
  return static_cast<const char*>(q.x) + (b * q.sb + s * q.ss) * SIZE<DT>;
}

// The logits' gradient, rows placed as the logits' are with strides of its own.
struct Grad {
  void* x;
  int64_t sb, ss;
};
template <int DT>
__device__ __forceinline__ char* grad_at(const Grad& g, int S, int64_t r) {
  const uint32_t b = (uint32_t)r / (uint32_t)S, s = (uint32_t)r - b * S;
  return static_cast<char*>(g.x) + (b * g.sb + s * g.ss) * SIZE<DT>;
}

constexpr int NT = 512;

struct LogpOut {
  double* logp64;  // any but logp may be null
  float* logp;
  float* entropy;
  RowStat* stat;
};

template <int DT, bool ENT>
__device__ __forceinline__ void write_logp(const LogpOut& o, int64_t r, const void* row,
                                           const Rows& q, const Joined& j, const RowStat& st) {
  const double lp =
      LN2 * (id_exponent(row_at_id<DT>(row, q.ids[r], q.V), q, j, st.m) - log2(j.S));
  if (o.logp64) o.logp64[r] = lp;
  o.logp[r] = (float)lp;
  if (ENT) o.entropy[r] = (float)(LN2 * (log2(j.S) - j.t / j.S));
  if (o.stat) o.stat[r] = st;
}
template <bool ENT>
__device__ __forceinline__ void write_uncounted(const LogpOut& o, int64_t r) {
  if (o.logp64) o.logp64[r] = 0.0;
  o.logp[r] = 0.f;
  if (ENT) o.entropy[r] = 0.f;
  if (o.stat) o.stat[r] = RowStat{0.f, 1.f, 0.f, 0.f};
}

// One workgroup a row. ONCE: nobody reads the logits again soon, so they are loaded past the
// caches (3992 x 151936 bf16 155 us = 5.9 TB/s, 174 without; but a backward finds float32
// logits of 200 MB in the last-level cache: with it 96 us, 112 past it).
template <int DT, bool ENT, bool ONCE>
__global__ void __launch_bounds__(NT) logp_kernel(Rows q, LogpOut o) {
  __shared__ JoinSpace<NT> red;
  const int64_t r = blockIdx.x;
  if (q.mask && !q.mask[r]) {
    if (threadIdx.x == 0) write_uncounted<ENT>(o, r);
    return;
  }
  const void* row = row_at<DT>(q, r);
  const Span<DT> sp(row, q.V);
  Sums<ENT> s;
  add_span<DT, ENT, ONCE, NT>(sp, 0, sp.nvec, true, q, s);
  RowStat st;
  const Joined j = row_stat<DT, ENT, NT>(s, row, q, red, &st);
  if (threadIdx.x == 0) write_logp<DT, ENT>(o, r, row, q, j, st);
}

// Few rows: each cut over gridDim.y workgroups, whose sums are then joined.
struct Part {
  double S, t;
  float M, pad;
};

template <int DT, bool ENT, bool ONCE>
__global__ void __launch_bounds__(NT) logp_part_kernel(Rows q, Part* parts) {
  __shared__ JoinSpace<NT> red;
  const int64_t r = blockIdx.x;
  if (q.mask && !q.mask[r]) return;
  const Span<DT> sp(row_at<DT>(q, r), q.V);
  const int n = (int)gridDim.y, y = (int)blockIdx.y, per = (sp.nvec + n - 1) / n;
  Sums<ENT> s;
  add_span<DT, ENT, ONCE, NT>(sp, min(sp.nvec, y * per), min(sp.nvec, (y + 1) * per), y == 0, q, s);
  const Joined j = join<ENT, NT>(s, red);
  if (threadIdx.x == 0) parts[r * n + y] = Part{j.S, j.t, j.M, 0.f};
}

template <int DT, bool ENT>
__global__ void __launch_bounds__(NT) logp_join_kernel(Rows q, const Part* parts, int n,
                                                       LogpOut o) {
  __shared__ JoinSpace<NT> red;
  const int64_t r = blockIdx.x;
  if (q.mask && !q.mask[r]) {
    if (threadIdx.x == 0) write_uncounted<ENT>(o, r);
    return;
  }
  Sums<ENT> s;
  if ((int)threadIdx.x < n) {
    const Part p = parts[r * n + threadIdx.x];
    s.M = p.M;
    s.S = p.S;
    s.t = p.t;
  }
  const void* row = row_at<DT>(q, r);
  RowStat st;
  const Joined j = row_stat<DT, ENT, NT>(s, row, q, red, &st);
  if (threadIdx.x == 0) write_logp<DT, ENT>(o, r, row, q, j, st);
}

// One row's gradient: value(x) = -c / T e(x) / S, and c / T more at id.
struct RowGrad {
  float khi, klo, M, m, neg, c;
  int id;  // -1: outside the vocabulary
};

__device__ __forceinline__ RowGrad row_grad(const Rows& q, const RowStat& st, float c,
                                            int64_t id) {
  return RowGrad{q.khi, q.klo, st.M, st.m, -c / st.S, c, id >= 0 && id < q.V ? (int)id : -1};
}
__device__ __forceinline__ float grad_value(const RowGrad& g, float x) {
  return __builtin_amdgcn_exp2f(exponent(x, g.khi, g.klo, g.M)) * g.neg;
}
// ... of rows whose M is not finite
__device__ __forceinline__ float grad_plain(const RowGrad& g, float x) {
  return __builtin_amdgcn_exp2f((x - g.m) * g.khi) * g.neg;
}

// A vector of a row's gradient. For 16-bit results |neg| goes into the exponent, so a value
// takes one multiply-add, the exponential and half a conversion: 2^(x khi + base), base =
// log2 |neg| - M + klo (M / khi). base rounds at 2^-24 of its size, klo is applied at the row's
// top instead of at x: together below 2^-13 of a value while |M| < 1024, where half a step of
// float16 is 2^-12 to 2^-11 of it; rows beyond that go value by value.
struct VecGrad {
  float khi, klo, M, neg, base;
  uint32_t sign;
};
__device__ __forceinline__ VecGrad vec_grad(const RowGrad& g) {
  return VecGrad{g.khi, g.klo, g.M, g.neg,
                 __builtin_amdgcn_logf(fabsf(g.neg)) - fmaf(-g.klo, g.M / g.khi, g.M),
                 __float_as_uint(g.neg) >> 31 ? 0x80008000u : 0u};
}
template <int DT>
__device__ __forceinline__ uint4 grad_vector(const VecGrad& g, const uint4& v) {
  float f[PER<DT>];
  unpack<DT>(v, f);
#pragma unroll
  for (int j = 0; j < PER<DT>; ++j)
    f[j] = DT == F32 ? __builtin_amdgcn_exp2f(exponent(f[j], g.khi, g.klo, g.M)) * g.neg
                     : __builtin_amdgcn_exp2f(fmaf(f[j], g.khi, g.base));
  uint4 o = pack<DT>(f);
  if (DT != F32) o = make_uint4(o.x ^ g.sign, o.y ^ g.sign, o.z ^ g.sign, o.w ^ g.sign);
  return o;
}
// Whether grad_vector holds for a row.
template <int DT>
__device__ __forceinline__ bool by_vectors(const RowGrad& g) {
  return DT == F32 ? g.M < INFINITY : fabsf(g.M) < 1024.f;
}

__device__ __forceinline__ void store_stream(void* p, uint4 v) {
  __builtin_nontemporal_store(u32x4_t{v.x, v.y, v.z, v.w}, reinterpret_cast<u32x4_t*>(p));
}

template <int DT, int NT>
__device__ __forceinline__ void zero_row(void* out, int V) {
  const Span<DT> sp(out, V);
  char* const o = static_cast<char*>(out) + (int64_t)sp.head * SIZE<DT>;
  for (int i = threadIdx.x; i < sp.nvec; i += NT)
    store_stream(o + (int64_t)i * 16, make_uint4(0, 0, 0, 0));
  if ((int)threadIdx.x < sp.odd) store1<DT>(out, sp.odd_at(threadIdx.x), 0.f);
}

// Rows that cannot be stored 16 bytes at a time where they are loaded so, and rows whose M
// is not finite: value by value (50257 bf16 values a row: 2.0 times the time).
template <int DT, int NT>
__device__ __noinline__ void grad_by_value(RowGrad g, const void* row, void* out, int V) {
  for (int v = threadIdx.x; v < V; v += NT) {
    const float x = load1<DT>(row, v);
    const float y = g.M < INFINITY ? grad_value(g, x) : grad_plain(g, x);
    store1<DT>(out, v, v == g.id ? y + g.c : y);
  }
}

// grad[r][v] = coef[r] scale / T (1[v = id] - e_v / S); scale: a device scalar or null.
// skip_one: the gradient for scale 1 is there already.
template <int DT>
__global__ void __launch_bounds__(NT) logits_grad_kernel(Rows q, int R, const RowStat* stat,
                                                         const float* coef, const float* scale,
                                                         float inv_t, Grad grad, bool skip_one) {
  const float by = scale ? *scale : 1.f;
  if (skip_one && by == 1.f) return;
  const int y = (int)blockIdx.y, ny = (int)gridDim.y;
  for (int64_t r = blockIdx.x; r < R; r += gridDim.x) {
    char* const out = grad_at<DT>(grad, q.S, r);
    if (q.mask && !q.mask[r]) {
      if (!skip_one && y == 0) zero_row<DT, NT>(out, q.V);
      continue;
    }
    const void* row = row_at<DT>(q, r);
    const RowGrad g = row_grad(q, stat[r], coef[r] * by * inv_t, q.ids[r]);
    const Span<DT> sp(row, q.V);
    char* const o = out + (int64_t)sp.head * SIZE<DT>;
    if (!aligned16(o) || !by_vectors<DT>(g)) {
      if (y == 0) grad_by_value<DT, NT>(g, row, out, q.V);
      continue;
    }
    const int idv = (g.id - sp.head) / PER<DT>;  // id's vector, if it is in one
    const bool in_vec = g.id >= sp.head && g.id < sp.tail;
    const VecGrad vg = vec_grad(g);
    for (int i = y * NT + (int)threadIdx.x; i < sp.nvec; i += ny * NT) {
      store_stream(o + (int64_t)i * 16, grad_vector<DT>(vg, sp.vec[i]));
      // the same thread's store to the same place comes after
      if (in_vec && i == idv)
        store1<DT>(out, g.id, grad_value(g, load1<DT>(row, g.id)) + g.c);
    }
    if (y == 0 && (int)threadIdx.x < sp.odd) {
      const int v = sp.odd_at(threadIdx.x);
      const float d = grad_value(g, load1<DT>(row, v));
      store1<DT>(out, v, v == g.id ? d + g.c : d);
    }
  }
}

// ------------------------------------------------------------- policy loss --

// What a token counts, by sequence: with n_b counted tokens in sequence b, n in all and B'
// sequences with some, 1 / n, 1 / (n_b B') or 1 / denom.
__device__ __forceinline__ double token_weight(const Policy& p, int in_row, double tokens,
                                               double seqs) {
  if (p.normalizer == 0) return 1.0 / tokens;
  if (p.normalizer == 1) return 1.0 / (in_row * seqs);
  return 1.0 / p.denom;
}

// Counted tokens of each sequence.
__global__ void __launch_bounds__(256) count_kernel(const uint8_t* mask, int S, int* counts) {
  __shared__ JoinSpace<256> red;
  const uint8_t* m = mask + (int64_t)blockIdx.x * S;
  int n = 0;
  for (int s = threadIdx.x; s < S; s += 256) n += m[s] != 0;
  const double all = block_sum64<256>((double)n, red);
  if (threadIdx.x == 0) counts[blockIdx.x] = (int)all;
}

// A batch of at most SMALL_TOKENS tokens in SMALL_BATCH sequences is counted by one workgroup,
// in its LDS: one launch instead of two.
constexpr int SMALL_BATCH = 1024, SMALL_TOKENS = 4096;

// counts[b] for a small batch: 64 positions a wave, one addition for them where they are of
// one sequence.
template <int NT_>
__device__ __forceinline__ void count_small(const uint8_t* mask, int B, int S, int* counts) {
  for (int b = threadIdx.x; b < B; b += NT_) counts[b] = 0;
  __syncthreads();
  const int R = B * S, lane = threadIdx.x & 63;
  for (int r0 = (int)(threadIdx.x & ~63u); r0 < R; r0 += NT_) {
    const int r = r0 + lane;
    const bool on = r < R && mask[r];
    const int b0 = r0 / S;
    const uint64_t set = __ballot(on);
    if (min(r0 + 63, R - 1) / S == b0) {
      if (lane == 0) atomicAdd(&counts[b0], __popcll(set));
    } else if (on) {
      atomicAdd(&counts[r / S], 1);
    }
  }
  __syncthreads();
}

// Counted tokens and sequences of the batch, the same in every thread.
template <int NT_>
__device__ __forceinline__ void totals(const int* counts, int B, double* red, double* tokens,
                                       double* seqs) {
  double n = 0.0, q = 0.0;
  for (int b = threadIdx.x; b < B; b += NT_) {
    const int c = counts[b];
    n += c;
    q += c > 0;
  }
  n = wave_sum64(n);
  q = wave_sum64(q);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6] = n;
    red[NT_ / 64 + (threadIdx.x >> 6)] = q;
  }
  __syncthreads();
  n = q = 0.0;
  for (int w = 0; w < NT_ / 64; ++w) {
    n += red[w];
    q += red[NT_ / 64 + w];
  }
  *tokens = n;
  *seqs = q;
}

// weights[b] of each sequence, and weights[B] = n, for the launches that follow.
template <bool SMALL>
__global__ void __launch_bounds__(1024) weight_kernel(Policy p, const uint8_t* mask, int B, int S,
                                                      const int* counts, double* weights) {
  __shared__ double red[2 * 16];
  __shared__ int own[SMALL ? SMALL_BATCH : 1];
  if (SMALL) count_small<1024>(mask, B, S, own);
  const int* const n = SMALL ? own : counts;
  double tokens, seqs;
  totals<1024>(n, B, red, &tokens, &seqs);
  for (int b = threadIdx.x; b < B; b += 1024) weights[b] = token_weight(p, n[b], tokens, seqs);
  if (threadIdx.x == 0) weights[B] = tokens;
}

struct Tokens {
  const double* logp64;  // [R], or null
  const double2* parts;  // [R] (the token's exponent, S), or null: logp is made of them
  float* logp;           // [R]: read where both are null, written where parts are given
  const float* old;      // [R] or null: logp itself
  const float* ref;      // [R] or null
  const float* adv;      // [B], or [R] (adv_tokens)
  const uint8_t* mask;   // [R] or null
  const double* weights; // [B + 1], or null: no mask, all of `weight`
  double weight;
  int B, S;
  bool adv_tokens;
};

// Sums over the counted tokens: w l, then r, stopped tokens, KL and old - logp.
struct TokenSums {
  double v[5];
};

// One token of ratio r and eq = exp(ref - logp): d l / d logp. A KL term of weight 0 is left
// out, not multiplied by it: eq may be infinite, and the reference be there for the metric alone.
struct Slope {
  double d, gain;
  bool follows;  // the smaller gain moves with r
};
__device__ __forceinline__ Slope token_slope(const Policy& p, double r, double a, bool has_ref,
                                             double eq) {
  const double lo = 1.0 - p.eps_low, hi = 1.0 + p.eps_high;
  const double clipped = fmin(fmax(r, lo), hi);
  const double free_gain = fmin(r, p.delta) * a, clip_gain = clipped * a;
  Slope s;
  s.follows = (free_gain <= clip_gain && r <= p.delta) ||
              (clip_gain <= free_gain && clipped == r);
  s.gain = fmin(free_gain, clip_gain);
  s.d = s.follows ? -r * a : 0.0;
  if (r != r || a != a) s.d = s.gain = r * a;  // fmin would hide a NaN
  if (has_ref && p.beta > 0.0) s.d += p.beta * (1.0 - eq);
  return s;
}

// Token r of sequence b and weight w: d loss / d logp, its terms added to s.
__device__ __forceinline__ double token_at(const Policy& p, const Tokens& t, int64_t r, int b,
                                           double lp, double w, TokenSums& s) {
  const double old = t.old ? (double)t.old[r] : lp, a = t.adv[t.adv_tokens ? r : b];
  const double ratio = exp(lp - old);
  double q = 0.0, eq = 1.0;
  if (t.ref) {
    q = (double)t.ref[r] - lp;
    eq = exp(q);
  }
  const Slope g = token_slope(p, ratio, a, t.ref != nullptr, eq);
  const double kl = t.ref ? eq - q - 1.0 : 0.0;
  s.v[0] += w * ((p.beta > 0.0 ? p.beta * kl : 0.0) - g.gain);
  s.v[1] += ratio;
  s.v[2] += g.follows ? 0.0 : 1.0;
  s.v[3] += kl;
  s.v[4] += old - lp;
  return g.d * w;
}

// The workgroup's sums, in wave order (thread 0 writes them).
template <int NT_>
__device__ __forceinline__ void write_sums(TokenSums s, double* red, double* out) {
#pragma unroll
  for (int i = 0; i < 5; ++i) s.v[i] = wave_sum64(s.v[i]);
  __syncthreads();
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int i = 0; i < 5; ++i) red[5 * (threadIdx.x >> 6) + i] = s.v[i];
  __syncthreads();
  if (threadIdx.x < 5) {
    double v = red[threadIdx.x];
    for (int w = 1; w < NT_ / 64; ++w) v += red[5 * w + threadIdx.x];
    out[threadIdx.x] = v;
  }
  __syncthreads();
}

// What the forward leaves for the backward: d loss / d logp of every token, 0 where not
// counted, in float64 (the log-probabilities' gradient) or float32 (the logits').
struct Coef {
  double* f64;
  float* f32;
};

struct LossOut {
  float* loss;
  float* metrics;
};

__device__ __forceinline__ void write_loss(const LossOut& o, const double* sums, double tokens) {
  *o.loss = (float)sums[0];
  for (int j = 0; j < 4; ++j) o.metrics[j] = tokens > 0.0 ? (float)(sums[1 + j] / tokens) : 0.f;
}

// ONE: a small batch by one workgroup, to the loss (and from the counts, without weights).
template <bool ONE, int NT_>
__global__ void __launch_bounds__(NT_) policy_kernel(Policy p, Tokens t, Coef coef, double* sums,
                                                     LossOut o) {
  __shared__ double red[5 * (NT_ / 64)], all[5];
  __shared__ int own[ONE ? SMALL_BATCH : 1];
  const int64_t R = (int64_t)t.B * t.S;
  const bool count = ONE && t.mask && !t.weights;
  double tokens = R, seqs = t.B;
  if (count) {
    count_small<NT_>(t.mask, t.B, t.S, own);
    totals<NT_>(own, t.B, red, &tokens, &seqs);
  } else if (t.weights) {
    tokens = t.weights[t.B];
  }
  TokenSums s{};
  for (int64_t r = (int64_t)blockIdx.x * NT_ + threadIdx.x; r < R; r += (int64_t)gridDim.x * NT_) {
    double d = 0.0;
    if (!t.mask || t.mask[r]) {
      const int b = (int)((uint32_t)r / (uint32_t)t.S);  // < 2^31 tokens
      const double w = count ? token_weight(p, own[b], tokens, seqs)
                       : t.weights ? t.weights[b] : t.weight;
      double lp;
      if (t.parts) {
        const double2 e = t.parts[r];
        lp = LN2 * (e.x - log2(e.y));
        t.logp[r] = (float)lp;
      } else {
        lp = t.logp64 ? t.logp64[r] : (double)t.logp[r];
      }
      d = token_at(p, t, r, b, lp, w, s);
    } else if (t.parts) {
      t.logp[r] = 0.f;
    }
    if (coef.f64) coef.f64[r] = d;
    if (coef.f32) coef.f32[r] = (float)d;
  }
  write_sums<NT_>(s, red, ONE ? all : sums + 5 * (int64_t)blockIdx.x);
  if (ONE && threadIdx.x == 0) write_loss(o, all, tokens);
}

// loss and metrics from the workgroups' sums, in their order.
__global__ void __launch_bounds__(256) finish_kernel(Tokens t, const double* sums, int blocks,
                                                     LossOut o) {
  __shared__ double red[20], all[5];
  TokenSums s{};
  for (int i = threadIdx.x; i < blocks; i += 256)
    for (int j = 0; j < 5; ++j) s.v[j] += sums[5 * i + j];
  write_sums<256>(s, red, all);
  if (threadIdx.x == 0) write_loss(o, all, t.weights ? t.weights[t.B] : (double)t.B * t.S);
}

// grad[r] = coef[r] * *by
__global__ void __launch_bounds__(256) scale_kernel(const double* coef, const float* by, int64_t n,
                                                    float* grad) {
  const double f = *by;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    grad[i] = (float)(coef[i] * f);
}

// ------------------------------------------- loss and gradient in one pass --

// A row of logits stays in registers from its sums to its gradient, so it is read once:
// NV vectors a thread, one row a workgroup. Between the sums and the gradient every wave but
// one waits, so that stretch is kept short: the token's inputs are loaded with the row, the
// ratio and exp(ref - logp) are made of the token's exponent and S without a logarithm, and
// logp itself is left to policy_kernel.
//
// REST: a row that does not fit into registers (19 vectors a thread, 311296 bytes). What is
// left is read again for the gradient and found in the last-level cache, since 256 rows are
// under way, a CU each, and 256 MB hold 1 MB of each: 2048 x 151936 float32 477 us, 5.2 TB/s of
// logits and gradient, where a pass for the sums and one for the gradient took 680.
template <int DT, int NT_, int NV, bool REST>
__global__ void __launch_bounds__(NT_, 4) loss_rows_kernel(Rows q, Policy p, Tokens t,
                                                           float inv_t, double2* parts,
                                                           RowStat* stat, float* coef,
                                                           Grad grad) {
  __shared__ JoinSpace<NT_> red;
  __shared__ RowGrad shared_grad;
  const uint32_t r = blockIdx.x;
  const int tid = threadIdx.x;
  char* const out = grad_at<DT>(grad, q.S, r);
  if (q.mask && !q.mask[r]) {
    zero_row<DT, NT_>(out, q.V);
    if (tid == 0) {
      stat[r] = RowStat{0.f, 1.f, 0.f, 0.f};
      coef[r] = 0.f;
    }
    return;
  }
  const void* row = row_at<DT>(q, r);
  const Span<DT> sp(row, q.V);
  // Stride i of the workgroup holds vectors start(i) + tid; the last one is moved back to end
  // with the row, and of it only what no stride before it holds counts (in_stride). So every
  // thread loads NV vectors in any case, at scalar addresses: were some loads skipped, the
  // compiler could not tell how many are behind the one it needs, and would wait for all.
  const int last = max(sp.nvec - NT_, 0), tail0 = min(tid, max(sp.nvec - 1, 0));
  auto start = [&](int i) __attribute__((always_inline)) {
    return REST ? i * NT_ : min(i * NT_, last);
  };
  auto in_stride = [&](int i) __attribute__((always_inline)) {
    return REST || (i ? tid >= i * NT_ - start(i) : tid < sp.nvec);
  };
  const uint4* const vec = REST || sp.nvec ? sp.vec : reinterpret_cast<const uint4*>(parts);
  uint4 v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i] = load_stream(vec + start(i) + tail0);
  // Loads come back in order: what is used before the row's last vector is loaded by scalar
  // loads, and what is a vector load is left as it stands (unconverted, and at an address
  // that looks as if it differed between lanes) until after the row's sums.
  int lane0 = 0;
  asm("" : "+v"(lane0));
  const int64_t id = load_uniform(q.ids + r);
  const bool known = id >= 0 && id < q.V;
  const Raw<DT> raw = load_raw<DT>(row, (known ? id : 0) + lane0);
  const Raw<DT> raw_odd = load_raw<DT>(row, tid < sp.odd ? sp.odd_at(tid) : 0);
  const uint32_t b = r / (uint32_t)t.S;
  const double adv = load_uniform(t.adv + (t.adv_tokens ? r : b));
  const double old = t.old ? (double)load_uniform(t.old + r) : 0.0;
  const double ref = t.ref ? (double)load_uniform(t.ref + r) : 0.0;
  const double w = t.weights ? load_uniform(t.weights + b) : t.weight;
  Sums<false> s;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (in_stride(i)) {
      float f[PER<DT>];
      unpack<DT>(v[i], f);
      s.admit(top_of<DT>(f), q);
      s.add(f, q);
    }
  }
  if (REST) add_span<DT, false, false, NT_, 4>(sp, NV * NT_, sp.nvec, false, q, s);
  const float odd = to_float<DT>(raw_odd);
  if (tid < sp.odd) {
    const float x[1] = {odd};
    s.admit(odd, q);
    s.add(x, q);
  }
  // by the first wave: d loss / d logp, and what the row's values need of it
  auto token = [&](const Joined& j, float m) __attribute__((always_inline)) {
    const float xid = known ? to_float<DT>(raw) : __builtin_nanf("");
    const double a = id_exponent(xid, q, j, m);
    const double ratio = t.old ? exp(fma(LN2, a, -old)) / j.S : 1.0 + 0.0 * a;
    const double eq = t.ref ? exp(fma(-LN2, a, ref)) * j.S : 1.0;
    const float c = (float)(token_slope(p, ratio, adv, t.ref != nullptr, eq).d * w);
    const RowStat st{j.M, (float)j.S, m, 0.f};
    if (tid == 0) {
      shared_grad = row_grad(q, st, c * inv_t, id);
      parts[r] = make_double2(a, j.S);
      stat[r] = st;
      coef[r] = c;
    }
  };
  leave<false, NT_>(s, red);
  __syncthreads();
  if (tid < 64) {
    const Joined j = gather<false, NT_>(red);
    if (usable(j)) token(j, 0.f);
    else if (tid == 0) shared_grad.neg = INFINITY, shared_grad.M = LOWEST;
  }
  __syncthreads();
  if (shared_grad.M == LOWEST) {  // no such row gets here through token()
    const PlainStat ps =
        plain_stat<DT, false, NT_>(row, q.V, q.khi, reinterpret_cast<float*>(&red));
    if (tid < 64) token(Joined{INFINITY, ps.S, 0.0}, ps.m);
    __syncthreads();
  }
  const RowGrad g = shared_grad;
  char* const o = out + (int64_t)sp.head * SIZE<DT>;
  if (!aligned16(o) || !by_vectors<DT>(g)) {
    grad_by_value<DT, NT_>(g, row, out, q.V);
    return;
  }
  const VecGrad vg = vec_grad(g);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (in_stride(i))
      store_stream(o + (int64_t)start(i) * 16 + tid * 16, grad_vector<DT>(vg, v[i]));
  }
  if (REST) {
    constexpr int AHEAD = 4;
    int i = NV * NT_ + tid;
    for (; i + (AHEAD - 1) * NT_ < sp.nvec; i += AHEAD * NT_) {
      uint4 u[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) u[k] = load_stream(sp.vec + i + k * NT_);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        store_stream(o + (int64_t)(i + k * NT_) * 16, grad_vector<DT>(vg, u[k]));
    }
    for (; i < sp.nvec; i += NT_)
      store_stream(o + (int64_t)i * 16, grad_vector<DT>(vg, load_stream(sp.vec + i)));
  }
  if (tid < sp.odd) {
    const int at = sp.odd_at(tid);
    const float y = grad_value(g, odd);
    store1<DT>(out, at, at == g.id ? y + g.c : y);
  }
  // the token's own value, by the thread that stored its vector (its later store to the
  // same place comes after)
  const int at_id = (g.id - sp.head) / PER<DT>;
  const int owner = REST ? at_id % NT_ : at_id - start(at_id / NT_);
  if (g.id >= sp.head && g.id < sp.tail && owner == tid)
    store1<DT>(out, g.id, grad_value(g, to_float<DT>(raw)) + g.c);
}

// ----------------------------------------------------------------- host --

// Workgroups a row of the log-probabilities is cut over: enough for 512 in all (two a CU; 8
// rows of 151936 bf16 logits 8.1 us, 17.3 with one workgroup each; with 1024 in all 200 rows
// gain 4 % and 32 lose 15), each with 1024 vectors or more (32 rows 8.5 us, 9.5 with 2048).
int logp_cuts(int64_t R, int dtype, int V) {
  const int64_t vecs = (int64_t)V * (dtype == F32 ? 4 : 2) / 16;
  const int64_t n = R ? (512 + R - 1) / R : 1;
  const int64_t most = vecs / 1024 < 64 ? vecs / 1024 : 64;
  return (int)(n < most ? n : most > 1 ? most : 1);
}
size_t logp_ws(int64_t R, int dtype, int V) {
  const int n = logp_cuts(R, dtype, V);
  return n > 1 ? (size_t)R * n * sizeof(Part) : 0;
}

// Workspace of the loss entry points: counts and weights per sequence, the workgroups' sums, and
// (from logits) the float64 log-probabilities and the parts of few rows.
constexpr int SUM_BLOCKS = 256;
struct PolicyWs {
  size_t counts, weights, sums, logp64, parts, total;
};
PolicyWs policy_ws(int B, int S, int dtype, int V) {  // V 0: from log-probabilities
  PolicyWs w{};
  size_t o = 0;
  auto take = [&](size_t n) {
    const size_t at = o;
    o += (n + 255) / 256 * 256;
    return at;
  };
  const int64_t R = (int64_t)B * S;
  w.counts = take((size_t)B * 4);
  w.weights = take((size_t)(B + 1) * 8);
  w.sums = take(SUM_BLOCKS * 5 * 8);
  w.logp64 = take(V ? (size_t)R * 16 : 0);  // or the parts that logp is made of
  w.parts = take(V ? logp_ws(R, dtype, V) : 0);
  w.total = o;
  return w;
}

int batch_check(int B, int S) {
  if (B < 0 || S < 0) return einval("negative dimension");
  if ((int64_t)B * S >= (1ll << 31) || B >= (1 << 23)) return einval("too many tokens");
  return GRPO_OK;
}

int rows_check(const void* x, int dtype, int64_t sb, int64_t ss, int B, int S, int V,
               const int64_t* ids, double temperature) {
  if (int rc = batch_check(B, S)) return rc;
  if ((int64_t)B * S >= (1 << 22)) return einval("2^22 rows of logits or more");
  if (V < 1) return einval("an empty vocabulary");
  // a thread's index and a stride beyond it stay ints
  if (V > 1 << 30) return einval("a vocabulary of more than 2^30 tokens");
  if (dtype < 0 || dtype > 2) return einval("dtype must be 0 (bf16), 1 (float16) or 2 (float32)");
  if (!(temperature > 0.0) || !(temperature < (double)INFINITY))
    return einval("temperature must be positive and finite");
  const float k = (float)(1.0 / LN2 / temperature);
  // (from 1e-20 on, what khi leaves of k is a normal float32 above 0)
  if (!(k >= 1e-20f) || !(k <= 1e30f)) return einval("temperature out of range");
  if ((int64_t)B * S == 0) return GRPO_OK;
  if (!x || !ids) return einval("null pointer");
  if (sb < 0 || ss < 0) return einval("negative row stride");
  const int size = dtype == F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(x) % size) return einval("logits are not aligned to their type");
  return GRPO_OK;
}

int grad_check(const void* grad, int dtype, int64_t sb, int64_t ss) {
  if (!grad) return einval("null pointer");
  if (sb < 0 || ss < 0) return einval("negative row stride");
  if (reinterpret_cast<uintptr_t>(grad) % (dtype == F32 ? 4 : 2))
    return einval("grad_logits is not aligned to its type");
  return GRPO_OK;
}

Rows rows_of(const void* x, int64_t sb, int64_t ss, int S, int V, const int64_t* ids,
             const uint8_t* mask, double temperature) {
  const double k = 1.0 / LN2 / temperature;
  float hi = (float)k;
  if ((double)hi >= k) hi = nextafterf(hi, 0.f);
  return Rows{x, sb, ss, S, V, ids, mask, k, hi, (float)(k - (double)hi)};
}

template <int DT, bool ENT, bool ONCE>
int launch_logp(const Rows& q, int64_t R, const LogpOut& o, Part* parts, hipStream_t st) {
  const int n = logp_cuts(R, DT, q.V);
  if (n == 1) {
    logp_kernel<DT, ENT, ONCE><<<(unsigned)R, NT, 0, st>>>(q, o);
    return launch_check("token_logprobs");
  }
  logp_part_kernel<DT, ENT, ONCE><<<dim3((unsigned)R, (unsigned)n), NT, 0, st>>>(q, parts);
  if (int rc = launch_check("token_logprobs_part")) return rc;
  logp_join_kernel<DT, ENT><<<(unsigned)R, NT, 0, st>>>(q, parts, n, o);
  return launch_check("token_logprobs_join");
}

// The last-level cache, which a backward may find its logits in.
constexpr int64_t CACHE = 256 << 20;

int run_logp(int dtype, const Rows& q, int64_t R, const LogpOut& o, void* parts, hipStream_t st) {
  Part* const p = static_cast<Part*>(parts);
  const bool once = !o.stat || R * q.V * (dtype == F32 ? 4 : 2) > CACHE;
  auto go = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (o.entropy)
      return once ? launch_logp<DT, true, true>(q, R, o, p, st)
                  : launch_logp<DT, true, false>(q, R, o, p, st);
    return once ? launch_logp<DT, false, true>(q, R, o, p, st)
                : launch_logp<DT, false, false>(q, R, o, p, st);
  };
  if (dtype == BF16) return go(std::integral_constant<int, BF16>{});
  if (dtype == F16) return go(std::integral_constant<int, F16>{});
  return go(std::integral_constant<int, F32>{});
}

int64_t row_vectors(int dtype, int V) { return ((int64_t)V * (dtype == F32 ? 4 : 2) + 15) / 16; }
int run_grad(int dtype, const Rows& q, int64_t R, const RowStat* stat, const float* coef,
             const float* scale, double temperature, const Grad& grad, bool skip_one, hipStream_t st) {
  const float inv_t = (float)(1.0 / temperature);
  const int n = (int)R;
  // with a gradient that is most likely there already, few workgroups to find that out; fewer
  // than 4096 rows are cut over several, of 1024 vectors or more each (993 x 50257 float32: 59
  // us with one each, 53)
  const int64_t cuts = std::min<int64_t>(4096 / n, row_vectors(dtype, q.V) / 1024);
  const dim3 grid(skip_one && n > 1024 ? 1024u : (unsigned)n, cuts > 1 ? (unsigned)cuts : 1u);
  if (dtype == BF16)
    logits_grad_kernel<BF16><<<grid, NT, 0, st>>>(q, n, stat, coef, scale, inv_t, grad, skip_one);
  else if (dtype == F16)
    logits_grad_kernel<F16><<<grid, NT, 0, st>>>(q, n, stat, coef, scale, inv_t, grad, skip_one);
  else
    logits_grad_kernel<F32><<<grid, NT, 0, st>>>(q, n, stat, coef, scale, inv_t, grad, skip_one);
  return launch_check("token_logprobs_backward");
}

// Whether loss and gradient are made by a workgroup a row. Few long rows are cut over the chip
// instead, for the sums and then for the gradient; us with a workgroup a row / with rows cut:
//   50257 float32     4 rows 15 / 17, 64 rows 15 / 16, 192 rows 22 / 26
//   151936 bfloat16   4 rows 23 / 16, 64 rows 24 / 19, 128 rows 25 / 27, 192 rows 30 / 38
//   151936 float32    64 rows 28 / 24, 128 rows 40 / 43, 512 rows 125 / 173, 2048 rows 477 / 680
//   262144 bfloat16   128 rows 45 / 41, 256 rows 66 / 72, 2048 rows 453 / 586
bool by_rows(int dtype, int64_t R, int V) {
  return row_vectors(dtype, V) <= 14 * 1024 || R >= 128;
}

template <int DT>
int launch_loss_rows(const Rows& q, int64_t R, const Policy& p, const Tokens& t, float inv_t,
                     double2* parts, RowStat* stat, float* coef, const Grad& grad, hipStream_t st) {
  const int64_t vecs = row_vectors(DT, q.V);
  auto go = [&](auto threads, auto each, auto rest) {
    constexpr int NT_ = decltype(threads)::value, NV = decltype(each)::value;
    constexpr bool REST = decltype(rest)::value;
    if (!REST && vecs > NT_ * NV) return false;
    loss_rows_kernel<DT, NT_, NV, REST>
        <<<(unsigned)R, NT_, 0, st>>>(q, p, t, inv_t, parts, stat, coef, grad);
    return true;
  };
  const std::integral_constant<int, 256> n256;
  const std::integral_constant<int, 512> n512;
  const std::integral_constant<int, 1024> n1024;
  const std::integral_constant<int, 10> v10;
  const std::integral_constant<int, 14> v14;
  const std::integral_constant<int, 19> v19;
  const std::integral_constant<int, DT == F32 ? 16 : 10> some;
  const std::false_type whole;
  // the smallest of these that holds the row (loads past it are loads all the same), or the
  // one that reads what it cannot hold twice, with registers left to do so
  go(n256, v10, whole) || go(n256, v19, whole) || go(n512, v14, whole) || go(n512, v19, whole) ||
      go(n1024, v14, whole) || go(n1024, v19, whole) || go(n1024, some, std::true_type{});
  return launch_check("policy_loss_rows");
}

int policy_check(const grpo_policy_t* p, int B, int S, const float* adv, const void* ws,
                 size_t ws_bytes, const PolicyWs& need) {
  if (int rc = batch_check(B, S)) return rc;
  if (!p) return einval("null policy parameters");
  if (!(p->eps_low >= 0.0) || !(p->eps_high >= 0.0)) return einval("clip range must be >= 0");
  if (!(p->delta > 0.0)) return einval("delta must be positive (infinity: no cap)");
  if (!(p->beta >= 0.0) || !(p->beta < INFINITY)) return einval("beta must be >= 0 and finite");
  if (p->normalizer < 0 || p->normalizer > 2) return einval("unknown normalizer");
  if (p->normalizer == 2 && !(p->denom > 0.0)) return einval("the normalizer must be positive");
  if ((int64_t)B * S && !adv) return einval("null pointer");
  if (!ws || (reinterpret_cast<uintptr_t>(ws) & 15u))
    return einval("the workspace must be 16-byte aligned");
  if (ws_bytes < need.total) {
    set_error("workspace too small");
    return GRPO_EWORKSPACE;
  }
  return GRPO_OK;
}

// Whether one workgroup ends a batch of up to `most` tokens; its counts have room for
// SMALL_BATCH sequences, of which there may be more than tokens (S = 0).
bool small_batch(const Tokens& t, int64_t most = SMALL_TOKENS) {
  return (int64_t)t.B * t.S <= most && t.B <= SMALL_BATCH;
}

// The weights for the launches that follow.
int run_weights(const Policy& p, Tokens* t, char* ws, const PolicyWs& o, hipStream_t st) {
  const double R = (double)t->B * t->S;
  t->weight = p.normalizer == 0 ? 1.0 / R : p.normalizer == 1 ? 1.0 / R : 1.0 / p.denom;
  if (!t->mask || R == 0.0) return GRPO_OK;
  int* const counts = reinterpret_cast<int*>(ws + o.counts);
  double* const weights = reinterpret_cast<double*>(ws + o.weights);
  t->weights = weights;
  if (small_batch(*t)) {
    weight_kernel<true><<<1, 1024, 0, st>>>(p, t->mask, t->B, t->S, nullptr, weights);
    return launch_check("policy_weights");
  }
  count_kernel<<<(unsigned)t->B, 256, 0, st>>>(t->mask, t->S, counts);
  if (int rc = launch_check("policy_count")) return rc;
  weight_kernel<false><<<1, 1024, 0, st>>>(p, t->mask, t->B, t->S, counts, weights);
  return launch_check("policy_weights");
}

// The tokens' losses and derivatives, and the sums' end; `one`: by one workgroup.
int run_policy(const Policy& p, const Tokens& t, bool one, char* ws, const PolicyWs& o, Coef coef,
               const LossOut& out, hipStream_t st) {
  const int64_t R = (int64_t)t.B * t.S;
  double* sums = reinterpret_cast<double*>(ws + o.sums);
  if (one) {
    policy_kernel<true, 1024><<<1, 1024, 0, st>>>(p, t, coef, sums, out);
    return launch_check("policy_loss");
  }
  const int64_t most = R ? cdiv(R, 256) : 1;
  const int blocks = (int)(most < SUM_BLOCKS ? most : SUM_BLOCKS);
  policy_kernel<false, 256><<<blocks, 256, 0, st>>>(p, t, coef, sums, out);
  if (int rc = launch_check("policy_loss")) return rc;
  finish_kernel<<<1, 256, 0, st>>>(t, sums, blocks, out);
  return launch_check("policy_finish");
}

}  // namespace

extern "C" size_t grpo_token_logprobs_workspace_bytes(int dtype, int B, int S, int V) {
  return dtype < 0 || dtype > 2 || B < 0 || S < 0 || V < 1 ? 0 : logp_ws((int64_t)B * S, dtype, V);
}

extern "C" int grpo_token_logprobs(const void* logits, int dtype, int64_t stride_b,
                                   int64_t stride_s, int B, int S, int V, const int64_t* ids,
                                   const uint8_t* mask, double temperature, float* logp,
                                   float* entropy, float* stat, void* workspace,
                                   size_t workspace_bytes, grpo_stream_t stream) {
  if (int rc = rows_check(logits, dtype, stride_b, stride_s, B, S, V, ids, temperature)) return rc;
  const int64_t R = (int64_t)B * S;
  if (!R) return GRPO_OK;
  if (!logp) return einval("null pointer");
  if (!aligned16(stat)) return einval("stat must be 16-byte aligned");
  if (const size_t need = logp_ws(R, dtype, V)) {
    if (!workspace || !aligned16(workspace)) return einval("the workspace must be 16-byte aligned");
    if (workspace_bytes < need) {
      set_error("workspace too small");
      return GRPO_EWORKSPACE;
    }
  }
  const LogpOut o{nullptr, logp, entropy, reinterpret_cast<RowStat*>(stat)};
  return run_logp(dtype, rows_of(logits, stride_b, stride_s, S, V, ids, mask, temperature), R, o,
                  workspace, as_stream(stream));
}

extern "C" int grpo_token_logprobs_backward(const void* logits, int dtype, int64_t stride_b,
                                            int64_t stride_s, int B, int S, int V,
                                            const int64_t* ids, const uint8_t* mask,
                                            double temperature, const float* stat,
                                            const float* grad_logp, const float* scale,
                                            void* grad_logits, int64_t grad_stride_b,
                                            int64_t grad_stride_s, grpo_stream_t stream) {
  if (int rc = rows_check(logits, dtype, stride_b, stride_s, B, S, V, ids, temperature)) return rc;
  const int64_t R = (int64_t)B * S;
  if (!R) return GRPO_OK;
  if (!stat || !grad_logp) return einval("null pointer");
  if (!aligned16(stat)) return einval("stat must be 16-byte aligned");
  if (int rc = grad_check(grad_logits, dtype, grad_stride_b, grad_stride_s)) return rc;
  return run_grad(dtype, rows_of(logits, stride_b, stride_s, S, V, ids, mask, temperature), R,
                  reinterpret_cast<const RowStat*>(stat), grad_logp, scale, temperature,
                  Grad{grad_logits, grad_stride_b, grad_stride_s}, false, as_stream(stream));
}

extern "C" size_t grpo_policy_loss_workspace_bytes(int B, int S) {
  return B < 0 || S < 0 ? 0 : policy_ws(B, S, 0, 0).total;
}

extern "C" int grpo_policy_loss(const float* logp, const float* old_logp, const float* ref_logp,
                                const float* advantages, int adv_tokens, const uint8_t* mask,
                                int B, int S, const grpo_policy_t* policy, float* loss,
                                float* metrics, double* coef, void* workspace,
                                size_t workspace_bytes, grpo_stream_t stream) {
  if (int rc = batch_check(B, S)) return rc;
  const PolicyWs o = policy_ws(B, S, 0, 0);
  if (int rc = policy_check(policy, B, S, advantages, workspace, workspace_bytes, o)) return rc;
  if (((int64_t)B * S && !logp) || !loss || !metrics) return einval("null pointer");
  Tokens t{nullptr, nullptr, const_cast<float*>(logp), old_logp, ref_logp, advantages, mask,
           nullptr, 0.0, B, S, adv_tokens != 0};
  hipStream_t st = as_stream(stream);
  char* const ws = static_cast<char*>(workspace);
  // one launch where it does (4096 tokens: 15 us of the GPU's time for 13 and a finish, and
  // 5 us less of the host's, which is what such a call waits for)
  const bool one = small_batch(t);
  if (!one || !mask) {
    if (int rc = run_weights(*policy, &t, ws, o, st)) return rc;
  }
  return run_policy(*policy, t, one, ws, o, Coef{coef, nullptr}, LossOut{loss, metrics}, st);
}

extern "C" int grpo_policy_loss_backward(const double* coef, const float* grad_loss,
                                         int64_t tokens, float* grad_logp, grpo_stream_t stream) {
  if (tokens < 0) return einval("negative dimension");
  if (!tokens) return GRPO_OK;
  if (!coef || !grad_loss || !grad_logp) return einval("null pointer");
  const int blocks = (int)(cdiv(tokens, 256) < 2048 ? cdiv(tokens, 256) : 2048);
  scale_kernel<<<blocks, 256, 0, as_stream(stream)>>>(coef, grad_loss, tokens, grad_logp);
  return launch_check("policy_loss_backward");
}

extern "C" size_t grpo_policy_loss_logits_workspace_bytes(int dtype, int B, int S, int V) {
  return dtype < 0 || dtype > 2 || B < 0 || S < 0 || V < 1 ? 0 : policy_ws(B, S, dtype, V).total;
}

extern "C" int grpo_policy_loss_logits(const void* logits, int dtype, int64_t stride_b,
                                       int64_t stride_s, int B, int S, int V, const int64_t* ids,
                                       const uint8_t* mask, double temperature,
                                       const float* old_logp, const float* ref_logp,
                                       const float* advantages, int adv_tokens,
                                       const grpo_policy_t* policy, float* loss, float* logp,
                                       float* metrics, float* stat, float* coef,
                                       void* grad_logits, int64_t grad_stride_b,
                                       int64_t grad_stride_s, void* workspace,
                                       size_t workspace_bytes, grpo_stream_t stream) {
  if (int rc = rows_check(logits, dtype, stride_b, stride_s, B, S, V, ids, temperature)) return rc;
  const PolicyWs o = policy_ws(B, S, dtype, V);
  if (int rc = policy_check(policy, B, S, advantages, workspace, workspace_bytes, o)) return rc;
  const int64_t R = (int64_t)B * S;
  if ((R && !logp) || !loss || !metrics) return einval("null pointer");
  if ((stat == nullptr) != (coef == nullptr)) return einval("stat and coef go together");
  if (!aligned16(stat)) return einval("stat must be 16-byte aligned");
  if (grad_logits && R && (!stat || !by_rows(dtype, R, V)))
    return einval("grad_logits needs stat and coef, and rows that are made in one pass");
  if (grad_logits) {
    if (int rc = grad_check(grad_logits, dtype, grad_stride_b, grad_stride_s)) return rc;
  }
  hipStream_t st = as_stream(stream);
  char* const ws = static_cast<char*>(workspace);
  double* const lp = reinterpret_cast<double*>(ws + o.logp64);
  RowStat* const rs = reinterpret_cast<RowStat*>(stat);
  Tokens t{lp, nullptr, logp, old_logp, ref_logp, advantages, mask, nullptr, 0.0, B, S,
           adv_tokens != 0};
  if (int rc = run_weights(*policy, &t, ws, o, st)) return rc;
  if (R) {
    const Rows q = rows_of(logits, stride_b, stride_s, S, V, ids, mask, temperature);
    const float inv_t = (float)(1.0 / temperature);
    int rc;
    if (!grad_logits) {
      rc = run_logp(dtype, q, R, LogpOut{lp, logp, nullptr, rs}, ws + o.parts, st);
    } else {
      auto go = dtype == BF16 ? launch_loss_rows<BF16>
                : dtype == F16 ? launch_loss_rows<F16> : launch_loss_rows<F32>;
      double2* const parts = reinterpret_cast<double2*>(lp);
      rc = go(q, R, *policy, t, inv_t, parts, rs, coef,
              Grad{grad_logits, grad_stride_b, grad_stride_s}, st);
      t.logp64 = nullptr;
      t.parts = parts;
      coef = nullptr;  // written
    }
    if (rc) return rc;
  }
  // one workgroup ends up to 1024 tokens (7.8 us), more are faster in two launches (10.6 at
  // 4096, one 16)
  return run_policy(*policy, t, small_batch(t, 1024), ws, o, Coef{nullptr, coef},
                    LossOut{loss, metrics}, st);
}

extern "C" int grpo_policy_loss_logits_one_pass(int dtype, int B, int S, int V) {
  return dtype >= 0 && dtype <= 2 && B >= 0 && S >= 0 && V >= 1 &&
         by_rows(dtype, (int64_t)B * S, V);
}

extern "C" int grpo_policy_loss_logits_rescale(const void* logits, int dtype, int64_t stride_b,
                                               int64_t stride_s, int B, int S, int V,
                                               const int64_t* ids, const uint8_t* mask,
                                               double temperature, const float* stat,
                                               const float* coef, const float* grad_loss,
                                               void* grad_logits, int64_t grad_stride_b,
                                               int64_t grad_stride_s, grpo_stream_t stream) {
  if (int rc = rows_check(logits, dtype, stride_b, stride_s, B, S, V, ids, temperature)) return rc;
  const int64_t R = (int64_t)B * S;
  if (!R) return GRPO_OK;
  if (!stat || !coef || !grad_loss) return einval("null pointer");
  if (!aligned16(stat)) return einval("stat must be 16-byte aligned");
  if (int rc = grad_check(grad_logits, dtype, grad_stride_b, grad_stride_s)) return rc;
  return run_grad(dtype, rows_of(logits, stride_b, stride_s, S, V, ids, mask, temperature), R,
                  reinterpret_cast<const RowStat*>(stat), coef, grad_loss, temperature,
                  Grad{grad_logits, grad_stride_b, grad_stride_s}, true, as_stream(stream));
}

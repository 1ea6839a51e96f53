// A token from each row of logits with temperature, top-k, top-p and min-p, from given
// uniform numbers (grpo_sample_tokens), without a sort. The place of the reference's _sample_tokens
// (src/triton_kernels/paged_kv.py:418-450) but not its top-p: the token at which the mass passes
// top_p is kept here, as the last of the shortest head that holds top_p of the mass, and cut there
// and in grpo_sample_top_p. Of .5, .3, .15, .05 at .9 three are kept here, two there.
//
// Row m: w_v = exp((x_v - max) / T), the row in descending order of x (ties by index). Kept
// is the head of that order with rank < k, then a mass before it below top_p times the mass
// of those k, then w >= min_p; the token is the first kept one at which the running mass
// passes u times the kept mass.
//
//  * Masses are integers, in units of 2^-S of the largest weight, S = 62 - ceil(log2 V), at most
//    44: their sums do not depend on the order in which threads add them, so the token is a
//    function of the inputs alone. Weights are doubles, rounded once to a unit where a bf16 row is
//    counted by its values; where bins of the distance stand for them, see there.
//  * "The first place in sorted order where the mass reaches P or the count reaches K" gives the
//    top-k, top-p and min-p cuts and the draw itself. It is found in a histogram of the row: of
//    its values in bf16, else of 4096 distances from the maximum and then, within the one of
//    them that holds the place, of the order-preserving keys until a bin is one value.
//
// A workgroup per row: of 1024 threads, or of 512 where there are more rows than CUs (two bf16 rows
// on a CU take turns at its atomics and its arithmetic: 512 x 151936 57 us against 70; 8 rows 29
// with 1024, 32 with 512) or where they are short.
#include <math.h>
#include <stddef.h>

#include <algorithm>

#include "scan.hpp"

using namespace grpo;

namespace {

struct TokArgs {
  const void* logits;
  int64_t ld;
  int M, V;
  const void* draws;
  int draws_f64;
  const float* temperature;  // per row, or null: t, k, p, mp for every row
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  double t, p, mp;
  int64_t k;
  int shift;  // S
  int64_t* tokens;
  int32_t* kept;
};

// Key of a logit: larger for a larger value, 0 for NaN and -inf. Float32 bits with the bits
// that the type never sets shifted out; -0 is +0.
template <int DT>
constexpr int LOW = DT == 0 ? 16 : (DT == 1 ? 13 : 0);
template <int DT>
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = x == 0.f ? 0u : __float_as_uint(x);
  const uint32_t o = b ^ ((b & 0x80000000u) ? 0xFFFFFFFFu : 0x80000000u);
  return x > -INFINITY ? o >> LOW<DT> : 0u;
}
template <int DT>
__device__ __forceinline__ float key_value(uint32_t k) {
  const uint32_t o = k << LOW<DT>;
  return (o & 0x80000000u) ? __uint_as_float(o ^ 0x80000000u)
                           : __uint_as_float(~o & ~((1u << LOW<DT>) - 1u));
}

template <int DT>
struct Elem {
  typedef uint16_t type;
  static constexpr int N = 8;
};
template <>
struct Elem<2> {
  typedef float type;
  static constexpr int N = 4;
};
template <int DT>
__device__ __forceinline__ float value_of(typename Elem<DT>::type x) {
  if constexpr (DT == 0) return bf2f(x);
  if constexpr (DT == 1) return h2f(x);
  if constexpr (DT == 2) return x;
}

// f(index, value as float) of every value of the row; 16-byte loads from the first boundary on.
template <int DT, int TT, typename F>
__device__ __forceinline__ void for_row(const typename Elem<DT>::type* row, int V, F&& f) {
  typedef typename Elem<DT>::type E;
  constexpr int N = Elem<DT>::N, U = 4;
  const int mis = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(E));
  const int head = min(V, mis ? N - mis : 0), G = (V - head) / N, tid = threadIdx.x;
  if (tid < head) f(tid, value_of<DT>(row[tid]));
  const E* const body = row + head;
#pragma unroll 1
  for (int g = tid; g < G; g += U * TT) {
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = *reinterpret_cast<const uint4*>(body + (int64_t)N * min(g + u * TT, G - 1));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (g + u * TT >= G) continue;
      const int at = head + N * (g + u * TT);
      const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (DT == 2) {
          f(at + e, __uint_as_float(w[e]));
        } else {
          f(at + 2 * e, value_of<DT>((uint16_t)w[e]));
          f(at + 2 * e + 1, value_of<DT>((uint16_t)(w[e] >> 16)));
        }
      }
    }
  }
  const int tail = head + N * G + tid;
  if (tail < V) f(tail, value_of<DT>(row[tail]));
}

// 2^-y as a double, y >= 0, times 2^up: Taylor polynomial of 2^f on [-1/2, 1/2], below 1e-14.
__device__ __forceinline__ double exp2_neg(double y, int up) {
  const double n = rint(y), f = n - y;
  double p = 4.44553827187081e-10;  // ln(2)^k / k!, k = 11 .. 0
  p = fma(p, f, 7.054911620801121e-09);
  p = fma(p, f, 1.0178086009239696e-07);
  p = fma(p, f, 1.3215486790144305e-06);
  p = fma(p, f, 1.5252733804059838e-05);
  p = fma(p, f, 0.00015403530393381606);
  p = fma(p, f, 0.0013333558146428441);
  p = fma(p, f, 0.009618129107628477);
  p = fma(p, f, 0.055504108664821576);
  p = fma(p, f, 0.2402265069591007);
  p = fma(p, f, 0.6931471805599453);
  p = fma(p, f, 1.0);
  return ldexp(p, up - (int)n);
}
// A double in [0, 2^52) as the nearest integer: its last place is 1 after 2^52 is added.
__device__ __forceinline__ uint64_t nearest(double x) {
  return (uint64_t)__double_as_longlong(x + 4503599627370496.0) & ((1ull << 52) - 1);
}
// A weight in units of 2^-shift (at most 2^-44); nothing more than shift + 1 doublings below the
// maximum.
__device__ __forceinline__ uint64_t mass_of(double y, int shift) {
  return y < (double)(shift + 1) ? nearest(exp2_neg(y, shift)) : 0;
}

// Distance from the maximum in doublings: 0 at the maximum itself (an infinite one included),
// infinite for what has no mass beside it.
struct Scale {
  double top, c;  // the maximum, log2(e) / T
  __device__ __forceinline__ double below(float x) const {
    const double y = (top - (double)x) * c;
    return x == (float)top ? 0.0 : (y >= 0.0 ? y : (double)INFINITY);
  }
};

// A row's settings. K: how many tokens top_k leaves; greedy: the maximum is taken.
struct Row {
  double T, p, mp;
  uint32_t K;
  bool greedy;
  uint64_t u;  // the draw in units of 2^-64
};
__device__ __forceinline__ Row row_of(const TokArgs& a, int m, uint32_t valid) {
  Row r;
  r.T = a.temperature ? (double)a.temperature[m] : a.t;
  r.p = a.top_p ? (double)a.top_p[m] : a.p;
  r.mp = a.min_p ? (double)a.min_p[m] : a.mp;
  const int64_t k = a.top_k ? (int64_t)a.top_k[m] : a.k;
  r.K = k > 0 && k < (int64_t)valid ? (uint32_t)k : valid;
  r.greedy = !(r.T > 0.0) || r.p <= 0.0 || r.mp > 1.0 || r.K == 1;
  // Two logits of any type differ by 2^-149 or not at all, so from 1e-300 down every weight but
  // the maximum's is 0, and log2(e) / T times 64 would become infinite: NaN at the maximum.
  r.T = fmax(r.T, 1e-300);
  const double u = a.draws_f64 ? static_cast<const double*>(a.draws)[m]
                               : (double)static_cast<const float*>(a.draws)[m];
  r.u = u > 0.0 ? (u < 1.0 ? (uint64_t)(u * 18446744073709551616.0) : ~0ull) : 0;
  return r;
}
// ceil(p * mass), at least 1.
__device__ __forceinline__ uint64_t share_of(double p, uint64_t mass) {
  const uint64_t f = (uint64_t)(p * 18446744073709551616.0);
  return max((uint64_t)1, (uint64_t)__umul64hi(f, mass) + (f * mass ? 1 : 0));
}
// How many weights w > 0 reach P > 0, at most `most` of them.
__device__ __forceinline__ uint32_t weights_for(uint64_t P, uint64_t w, uint32_t most) {
  double q = (double)P / (double)w;
  if (!(q < (double)most)) return most;
  uint32_t n = (uint32_t)q;  // the quotient or a neighbour of it
  while (n && n * w >= P) --n;
  while (n * w < P) ++n;
  return min(n, most);
}

// Where a search ends: the value, the tokens before it in sorted order, how many of those that
// hold it are needed (1 or more), the mass up to the last of them.
struct Leaf {
  uint32_t key, before, in;
  uint64_t total;
};

// The cuts and the draw, from a search(P, K, more) for the first place where the mass reaches P
// (0: no such bound) or the count K (more: others follow); `near` tokens pass min_p, `all` is the
// row's mass.
template <typename Search>
__device__ __forceinline__ Leaf draw_of(const Row& r, uint32_t valid, uint32_t near, uint64_t all,
                                        uint32_t& kept, Search&& search) {
  const uint32_t K = r.mp > 0.0 ? min(r.K, max(near, 1u)) : r.K;
  uint64_t mass = r.K < valid && r.p < 1.0 ? 0 : all;  // of what top_k leaves; then of what is kept
  kept = valid;
  Leaf l;
  // (one place that calls it: the code is large, and runs at the rate of its instruction
  // fetches the first time)
#pragma unroll 1
  for (int stage = mass ? 1 : 0; stage < 3; ++stage) {
    const uint64_t P = stage == 0   ? 0
                       : stage == 2 ? __umul64hi(r.u, mass) + 1
                       : r.p < 1.0  ? share_of(r.p, mass)
                                    : 0;
    if (stage == 1 && !P && K >= valid) continue;
    l = search(P, stage == 0 ? r.K : stage == 1 ? K : kept, stage < 2);
    mass = l.total;
    if (stage == 1) kept = l.before + l.in;
  }
  return l;
}
__device__ __forceinline__ bool reached(uint64_t mass, uint32_t count, uint64_t P, uint32_t K) {
  return (P && mass >= P) || count >= K;
}

struct Found {
  uint64_t mass, own;  // before the bin, of the bin
  uint32_t bin, before, group;
};
struct Slots {
  uint64_t s64[16];  // (the scans read a row of lanes of them)
  uint32_t s32[16];
  Found found;
  Leaf leaf;
  uint32_t n_list, best, range[2];
};

// First index of the value with key `key` (all threads get it).
template <int DT, int TT>
__device__ __forceinline__ uint32_t first_index(const typename Elem<DT>::type* row, int V,
                                                uint32_t key, Slots& s) {
  if (threadIdx.x == 0) s.best = 0xFFFFFFFFu;
  __syncthreads();
  const float x = key_value<DT>(key);  // (-0 is equal to it too)
  uint32_t best = 0xFFFFFFFFu;
  for_row<DT, TT>(row, V, [&](int i, float v) { best = v == x ? min(best, (uint32_t)i) : best; });
  if (best != 0xFFFFFFFFu) atomicMin(&s.best, best);
  __syncthreads();
  return s.best;
}

template <int DT, int TT>
__device__ __forceinline__ void maximum(const typename Elem<DT>::type* row, int V, uint32_t& kmax,
                                        uint32_t& valid, Slots& s) {
  float top = -INFINITY;
  uint32_t n = 0;
  for_row<DT, TT>(row, V, [&](int, float x) {
    top = fmaxf(top, x);
    n += x > -INFINITY ? 1u : 0u;
  });
  kmax = block_max<TT / 64>(key_of<DT>(top), s.s32);
  valid = block_sum<TT / 64>(n, s.s32);
}

// Rows with nothing to draw, or whose maximum is taken; true if done.
template <int DT, int TT>
__device__ __forceinline__ bool simple_row(const TokArgs& a, int m, uint32_t kmax, const Row& r,
                                           Slots& s) {
  typedef typename Elem<DT>::type E;
  if (kmax && !r.greedy) return false;
  int64_t token = -1;
  if (kmax)
    token = first_index<DT, TT>(static_cast<const E*>(a.logits) + (int64_t)m * a.ld, a.V, kmax, s);
  if (threadIdx.x == 0) {
    a.tokens[m] = token;
    if (a.kept) a.kept[m] = kmax ? 1 : 0;
  }
  return true;
}

// ------------------------------------------------- bins of the distance --
// 64 bins per doubling below the maximum. A token adds one 64-bit number to its bin: 1 to the
// count in the upper bits, and (1 - 2^-(f / 64)) 2^UNIT to a sum in the lower ones, f its place in
// the bin. A bin's mass is 2^-(bin / 64) (count - sum): one LDS atomic and 4 FMAs per token
// instead of two and an exponential. A token's weight in it is off by 1.3e-12 of itself at most for
// the series and half a unit for its place: 2^-(71 - 2 bits of V), 2e-12 up to 65535 tokens, 3e-11
// up to 262143, 2e-9 for 2^20. Within a bin the tokens' weights are relative to the bin's first
// (2^-44), and P is a share of the bin's mass.
constexpr int NB = 4096;
constexpr int LIST = 4096;     // tokens of one bin that LDS holds
constexpr int ALL = 1024;      // of all bins down to one (512 to 4096: no difference)
constexpr double A64 = 0.010830424696249145;  // ln(2) / 64

template <int TT>
struct General {
  unsigned long long bins[NB];
  unsigned long long kmass[TT];  // bins of keys, one per thread
  uint32_t kcnt[TT];
  uint32_t lkey[LIST];
  uint32_t lidx[LIST];
  Slots s;
};

__device__ __forceinline__ double bin_place(double y) { return fmin(y * 64.0, (double)(NB - 1)); }

// Smallest key in [1, kmax] whose bin is at most j: 64 candidates at a time, by one wave.
template <int DT>
__device__ __forceinline__ uint32_t first_key(const Scale& sc, uint32_t kmax, int j) {
  uint32_t lo = 1, hi = kmax;  // hi holds
#pragma unroll 1
  while (lo < hi) {
    const uint32_t step = (hi - lo) / 64 + 1, lane = threadIdx.x & 63;
    const uint32_t c = (uint32_t)min((uint64_t)lo + (uint64_t)lane * step, (uint64_t)hi);
    const uint64_t is = __ballot((int)bin_place(sc.below(key_value<DT>(c))) <= j);
    const uint32_t f = is ? __builtin_ctzll(is) : 64;
    const uint32_t at = lo;
    if (f < 64) hi = (uint32_t)min((uint64_t)at + (uint64_t)f * step, (uint64_t)hi);
    lo = f ? at + (f - 1) * step + 1 : hi;
  }
  return hi;
}

template <int DT, int TT>
__device__ __forceinline__ void general_row(const TokArgs& a, int m, General<TT>& s, uint32_t kmax,
                                            uint32_t valid, const Row& r) {
  typedef typename Elem<DT>::type E;
  constexpr int PER = NB / TT, KEY_BITS = TT == 1024 ? 10 : 9;
  static_assert(TT == 1 << KEY_BITS, "a bin of keys per thread");
  const int tid = threadIdx.x, V = a.V, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const E* const row = static_cast<const E*>(a.logits) + (int64_t)m * a.ld;
  const Scale sc{key_value<DT>(kmax), 1.4426950408889634 / r.T};
  const double ymin = r.mp > 0.0 ? -log2(r.mp) : INFINITY;
  // The sum of V places, below V A64 2^unit, stays in the lower bits, their count in the upper
  // (13 at least: a place of 2^-44 is as fine as a mass).
  const int cbits = max(13, 32 - __clz(V)), unit = 70 - 2 * cbits, sbits = 64 - cbits;
  for (int j = tid; j < NB; j += TT) s.bins[j] = 0;
  __syncthreads();
  uint32_t near = 0;  // tokens that min_p leaves
  {
    const double sl = ldexp(1.0, unit), k1 = A64 * sl, k2 = -A64 * A64 / 2 * sl,
                 k3 = A64 * A64 * A64 / 6 * sl, k4 = -A64 * A64 * A64 * A64 / 24 * sl;
    auto add = [&](double z) {
      near += z <= ymin * 64.0 ? 1u : 0u;
      z = fmin(z, (double)(NB - 1));
      const int b = (int)z;
      const double f = z - b;
      const uint64_t place = nearest(f * fma(fma(fma(k4, f, k3), f, k2), f, k1));
      atomicAdd(&s.bins[b], (unsigned long long)(place + (1ull << sbits)));
    };
    if (valid == (uint32_t)V && sc.top < INFINITY) {
      const double c = sc.c * 64.0;
      for_row<DT, TT>(row, V, [&](int, float x) { add((sc.top - (double)x) * c); });
    } else {
      for_row<DT, TT>(row, V, [&](int, float x) {
        if (x > -INFINITY) add(sc.below(x) * 64.0);
      });
    }
  }
  if (r.mp > 0.0) near = block_sum<TT / 64>(near, s.s.s32);
  __syncthreads();
  // this thread's bins: masses, counts, and what stands before them
  uint64_t bm[PER], pm = 0;
  uint32_t bc[PER], pc = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const uint64_t v = s.bins[tid * PER + j];
    bc[j] = (uint32_t)(v >> sbits);
    const double part = (double)bc[j] - ldexp((double)(v & ((1ull << sbits) - 1)), -unit);
    bm[j] = bc[j] ? (uint64_t)rint(part * exp2_neg((tid * PER + j) * (1.0 / 64), a.shift)) : 0;
    pm += bm[j];
    pc += bc[j];
  }
  const uint64_t tm = pm;
  const uint32_t tc = pc;
  block_excl_scan(pm, pc, s.s.s64, s.s.s32);
  const uint64_t all = block_sum<TT / 64>(tm, s.s.s64);

  // The list holds the tokens of bins list0 to list1: of all down to a search's bin, if they are
  // few and searches follow (which end in or before it), else of that bin alone.
  int list0 = 0, list1 = -1, last = -1;  // last: the bin that held the last place
  auto search = [&](uint64_t P, uint32_t K, bool more) {
    if (P > all) P = all;
    if (!reached(pm, pc, P, K) && reached(pm + tm, pc + tc, P, K)) {
      uint64_t mj = pm;
      uint32_t cj = pc;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (!reached(mj, cj, P, K) && reached(mj + bm[j], cj + bc[j], P, K))
          s.s.found = Found{mj, bm[j], (uint32_t)(tid * PER + j), cj, bc[j]};
        mj += bm[j];
        cj += bc[j];
      }
    }
    __syncthreads();
    const Found top = s.s.found;
    const int bin = last = top.bin;
    const bool all_before = more && top.before + top.group <= ALL;
    bool list = bin >= list0 && bin <= list1;
    if (list) {  // the bin's keys
      if (tid < 2) s.s.range[tid] = tid ? 0u : 0xFFFFFFFFu;
      __syncthreads();
      for (uint32_t i = tid; i < min(s.s.n_list, (uint32_t)LIST); i += TT) {
        const uint32_t k = s.lkey[i];
        if ((int)bin_place(sc.below(key_value<DT>(k))) != bin) continue;
        atomicMin(&s.s.range[0], k);
        atomicMax(&s.s.range[1], k);
      }
    } else {
      if (wave < 2) {  // they are below the first one of the bin before
        const uint32_t k = bin >= wave ? first_key<DT>(sc, kmax, bin - wave) : kmax + 1;
        if ((tid & 63) == 0) s.s.range[wave] = k - wave;
      }
      if (tid == 0) s.s.n_list = 0;
      list0 = all_before ? 0 : bin;
      list1 = top.group <= LIST ? bin : -1;
    }
    __syncthreads();
    uint32_t lo = s.s.range[0], hi = s.s.range[1];
    if (!list && top.group <= LIST) {
      // (the last bin begins at a key of NaN)
      const float xlo = fmaxf(key_value<DT>(lo), -__FLT_MAX__);
      const float xhi = all_before ? INFINITY : key_value<DT>(hi);
      for_row<DT, TT>(row, V, [&](int i, float x) {
        if (!(x >= xlo && x <= xhi)) return;
        const uint32_t at = atomicAdd(&s.s.n_list, 1u);
        if (at >= LIST) return;  // (never: the bins hold as many)
        s.lkey[at] = key_of<DT>(x);
        s.lidx[at] = i;
      });
      list = true;
      __syncthreads();
    }
    const uint32_t n = min(s.s.n_list, (uint32_t)LIST);
    // weights relative to the bin's start: 2^44 of it at most
    auto rel = [&](uint32_t k) {
      const double y = sc.below(key_value<DT>(k)) - bin * (1.0 / 64);
      return nearest(exp2_neg(fmin(fmax(y, 0.0), 1000.0), a.shift));
    };
    // P among those, if it lies in this bin; a bin whose tokens have no mass of their own: all
    auto share = [&](uint64_t sum) -> uint64_t {
      if (!P || P > top.mass + top.own) return 0;
      const double x =
          top.own ? (double)(P - top.mass) / (double)top.own * (double)sum : (double)sum;
      return min(max((uint64_t)ceil(x), (uint64_t)1), max(sum, (uint64_t)1));
    };
    uint64_t Q = 0, mb = 0, sum = 0;  // P in those, before the range, of the whole bin
    uint32_t cb = top.before, group = top.group;
    bool first = true;
#pragma unroll 1
    while (lo < hi) {
      const int sh = max(0, 32 - __clz(hi - lo) - KEY_BITS);
      s.kmass[tid] = 0;
      s.kcnt[tid] = 0;
      __syncthreads();
      auto add = [&](uint32_t k) {
        if (k < lo || k > hi) return;
        atomicAdd(&s.kmass[(hi - k) >> sh], (unsigned long long)rel(k));
        atomicAdd(&s.kcnt[(hi - k) >> sh], 1u);
      };
      if (list) {
#pragma unroll 1
        for (uint32_t i = tid; i < n; i += TT) add(s.lkey[i]);
      } else {
        for_row<DT, TT>(row, V, [&](int, float x) { add(key_of<DT>(x)); });
      }
      __syncthreads();
      const uint64_t mt = s.kmass[tid];
      const uint32_t ct = s.kcnt[tid];
      uint64_t before = mt;
      uint32_t upto = ct;
      block_excl_scan(before, upto, s.s.s64, s.s.s32);
      if (first) {
        sum = block_sum<TT / 64>(mt, s.s.s64);
        Q = share(sum);
        first = false;
      }
      before += mb;
      upto += cb;
      if (!reached(before, upto, Q, K) && reached(before + mt, upto + ct, Q, K))
        s.s.found = Found{before, mt, (uint32_t)tid, upto, ct};
      __syncthreads();
      const Found f = s.s.found;
      const uint32_t q = min(f.bin, (hi - lo) >> sh), width = (1u << sh) - 1;
      mb = f.mass;
      cb = f.before;
      group = f.group;
      hi -= q << sh;
      if (hi - lo > width) lo = hi - width;
      __syncthreads();
      if (list && group == 1 && lo < hi) {  // the token itself
#pragma unroll 1
        for (uint32_t i = tid; i < n; i += TT)
          if (s.lkey[i] >= lo && s.lkey[i] <= hi) s.s.range[0] = s.lkey[i];
        __syncthreads();
        lo = hi = s.s.range[0];
      }
    }
    const uint64_t w = rel(hi);
    if (first) {  // the bin is one value
      sum = w * group;
      Q = share(sum);
    }
    Leaf l;
    l.key = hi;
    l.before = cb;
    l.in = min(group, K - cb);
    if (Q > mb && w) l.in = weights_for(Q - mb, w, l.in);
    l.in = max(l.in, 1u);
    const uint64_t end = mb + l.in * w;
    l.total = top.mass + (end >= sum ? top.own
                                     : (uint64_t)rint((double)end / (double)sum * (double)top.own));
    l.total = max(l.total, (uint64_t)1);
    return l;
  };

  uint32_t kept;
  const Leaf d = draw_of(r, valid, near, all, kept, search);
  // The token of rank d.in - 1 by index among those of this value: the segment of 2^seg tokens
  // that holds it, then the place in it.
  const int seg = max(0, 32 - __clz(V - 1) - KEY_BITS);
  s.kcnt[tid] = 0;
  __syncthreads();
  if (last >= list0 && last <= list1) {
#pragma unroll 1
    for (uint32_t i = tid; i < min(s.s.n_list, (uint32_t)LIST); i += TT)
      if (s.lkey[i] == d.key) atomicAdd(&s.kcnt[s.lidx[i] >> seg], 1u);
  } else {
    const float x = key_value<DT>(d.key);
    for_row<DT, TT>(row, V, [&](int i, float v) {
      if (v == x) atomicAdd(&s.kcnt[i >> seg], 1u);
    });
  }
  __syncthreads();
  const uint32_t rank = d.in - 1, mine = s.kcnt[tid];
  uint64_t unused = 0;
  uint32_t upto = mine;
  block_excl_scan(unused, upto, s.s.s64, s.s.s32);
  if (upto <= rank && rank < upto + mine) {
    s.s.found.bin = tid;
    s.s.found.before = upto;
  }
  __syncthreads();
  if (tid >= 64) return;
  const int i0 = (int)s.s.found.bin << seg, i1 = min(V, i0 + (1 << seg));
  uint32_t left = rank - s.s.found.before;
#pragma unroll 1
  for (int i = i0; i < i1; i += 64) {
    const int at = i + tid;
    const bool hit = at < i1 && key_of<DT>(value_of<DT>(row[min(at, V - 1)])) == d.key;
    const uint64_t hits = __ballot(hit);
    const uint32_t c = __popcll(hits);
    if (left < c) {
      if (hit && (uint32_t)__popcll(hits & ((1ull << tid) - 1)) == left) {
        a.tokens[m] = at;
        if (a.kept) a.kept[m] = (int32_t)kept;
      }
      return;
    }
    left -= c;
  }
}

template <int DT, int TT>
__global__ void __launch_bounds__(TT) sample_tokens_kernel(TokArgs a) {
  typedef typename Elem<DT>::type E;
  extern __shared__ __align__(16) char lds_raw[];
  General<TT>& s = *reinterpret_cast<General<TT>*>(lds_raw);
  const int m = blockIdx.x;
  uint32_t kmax, valid;
  maximum<DT, TT>(static_cast<const E*>(a.logits) + (int64_t)m * a.ld, a.V, kmax, valid, s.s);
  const Row r = row_of(a, m, valid);
  if (simple_row<DT, TT>(a, m, kmax, r, s.s)) return;
  general_row<DT, TT>(a, m, s, kmax, valid, r);
}

// ------------------------------------------------------- bf16: its values --
// A bf16 row has few distinct values: their counts, one 32-bit LDS atomic per token, and a
// weight per value. The bins are fixed, the values of magnitude 2^-30 to 512 (without) in
// descending order with one bin for 0 and what is smaller among them, so that one pass over the
// row makes the counts, which tell the maximum too. A row with smaller values than 2^-30 other
// than 0, with a larger maximum, or with mass at -512 and below (an extreme temperature) takes
// the bins of the distance. The second pass over the row looks for the token and ends where it is
// found.
// Bound on its CU by loading and counting (16 of 28 us at 151936 tokens; stores in place of the
// atomics take as long) and by the issue of what is done per token (1 us per instruction). (The row in registers instead of its second reading: 8 / 512
// rows 39 / 155 us, in code without loops that runs at the rate of its instruction fetches.)
constexpr int LEAST = 0x3080, LARGE = 0x4400;  // the bits of 2^-30 and 512
constexpr int ZERO = LARGE - LEAST + 1;        // bin of 0; 0 and 2 ZERO: from +-512 on
constexpr int CW = 64;                         // bins of a group: one per lane
constexpr int CG = (2 * ZERO + 1 + CW - 1) / CW;
constexpr int U16 = 5;                         // 16-byte groups in flight per thread
constexpr int SEGS = GRPO_SAMPLE_MAX_VOCAB / (8 * 64 * U16) + 17 + 2;
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

struct Counts {
  uint32_t n[CG * CW];
  uint64_t mass[CG + 1];  // of the groups
  uint32_t count[CG + 3]; // (all of these are zero at first)
  Slots s;
};
static_assert(offsetof(Counts, s) % 16 == 0, "cleared 16 bytes at a time");
static_assert(CG <= 512 && SEGS <= 512, "a group, a segment per thread");

__device__ __forceinline__ u16x2 bin_of(uint32_t pair) {
  const u16x2 x = __builtin_bit_cast(u16x2, pair);
  const u16x2 size = __builtin_elementwise_min(
      __builtin_elementwise_sub_sat((u16x2)(x & (uint16_t)0x7FFF), (u16x2)(uint16_t)(LEAST - 1)),
      (u16x2)(uint16_t)ZERO);
  const u16x2 sign = (x >> 15) * (uint16_t)2 - (uint16_t)1;  // -1 for what is positive
  return size * sign + (uint16_t)ZERO;
}
__device__ __forceinline__ uint32_t bin_bits(int bin) {
  const int size = bin < ZERO ? ZERO - bin : bin - ZERO;
  return size ? (uint32_t)(size + LEAST - 1) | (bin > ZERO ? 0x8000u : 0u) : 0u;
}

// Where the row's 16-byte groups begin, and how many they are. A wave takes 64 U16 neighbouring
// groups at a time (a segment), 64 of them by each load.
template <int TT>
struct Groups {
  const uint16_t* row;
  int V, head, G;
  __device__ __forceinline__ Groups(const TokArgs& a, int m)
      : row(static_cast<const uint16_t*>(a.logits) + (int64_t)m * a.ld), V(a.V) {
    const int mis = (int)((reinterpret_cast<uintptr_t>(row) & 15) / 2);
    head = min(V, mis ? 8 - mis : 0);
    G = (V - head) / 8;
  }
  __device__ __forceinline__ uint4 at(int g) const {
    return *reinterpret_cast<const uint4*>(row + head + 8 * (int64_t)min(g, G - 1));
  }
  // one(0 or 1, value) of the values before and after the groups, many(group), done(segment) of
  // all threads after each of its wave's segments; true ends it.
  template <typename One, typename Many, typename Done>
  __device__ __forceinline__ void each(One&& one, Many&& many, Done&& done) const {
    const int tid = threadIdx.x, tail = head + 8 * G + tid;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (tid < head) one(0, row[tid]);
    if (tail < V) one(1, row[tail]);
#pragma unroll 1
    for (int s = wave; s - wave < (G + 64 * U16 - 1) / (64 * U16); s += TT / 64) {
      const int g = 64 * U16 * s + (tid & 63);
      uint4 w[U16];
#pragma unroll
      for (int u = 0; u < U16; ++u) w[u] = at(g + 64 * u);
#pragma unroll
      for (int u = 0; u < U16; ++u)
        if (g + 64 * u < G) many(w[u]);
      if (done(s)) break;
    }
  }
};
struct Never {
  __device__ __forceinline__ bool operator()(int) const { return false; }
};

// The token of rank `rank` among those whose bits are want (two of them, compared in mask).
template <int TT>
__device__ __forceinline__ void pick_bits(const TokArgs& a, const Groups<TT>& x, int m,
                                          uint32_t want, uint32_t mask, uint32_t rank,
                                          uint32_t kept, Counts& s) {
  const int tid = threadIdx.x, lane = tid & 63;
  // segments: before the groups, the waves' (an unfinished round's too), after them
  const int segs = 2 + (x.G + 64 * U16 - 1) / (64 * U16) + TT / 64;
  if (tid < SEGS) s.n[tid] = 0;
  if (tid == 0) s.s.n_list = 0;
  __syncthreads();
  auto differ = [&](const uint4& w) {  // in the halves of the sum: how many of the values do
    const uint32_t p[4] = {w.x, w.y, w.z, w.w};
    u16x2 n = (uint16_t)0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      n += __builtin_elementwise_min(__builtin_bit_cast(u16x2, (p[i] ^ want) & mask),
                                     (u16x2)(uint16_t)1);
    return n;
  };
  auto is = [&](uint16_t v) { return ((v ^ want) & mask & 0xFFFFu) == 0; };
  u16x2 not_it = (uint16_t)0;
  uint32_t looked = 0;
  x.each(
      [&](int end, uint16_t v) {
        if (!is(v)) return;
        atomicAdd(&s.n[end ? segs - 1 : 0], 1u);
        if (!end) atomicAdd(&s.s.n_list, 1u);
      },
      [&](const uint4& w) {
        not_it += differ(w);
        looked += 8;
      },
      [&](int seg) {  // is the token among those looked at so far?
        const uint32_t c = wave_prefix(looked - not_it[0] - not_it[1], Add());
        if (lane == 63 && c) {
          s.n[1 + seg] = c;
          atomicAdd(&s.s.n_list, c);
        }
        not_it = (uint16_t)0;
        looked = 0;
        __syncthreads();
        const bool is_there = s.s.n_list > rank;
        __syncthreads();  // (read by all before more is added)
        return is_there;
      });
  __syncthreads();
  const uint32_t mine = tid < segs ? s.n[tid] : 0;
  uint32_t upto = mine;
  uint64_t unused = 0;
  block_excl_scan(unused, upto, s.s.s64, s.s.s32);
  if (upto <= rank && rank < upto + mine) {
    s.s.found.bin = tid;
    s.s.found.before = upto;
  }
  __syncthreads();
  if (tid >= 64) return;
  const int seg = (int)s.s.found.bin;
  uint32_t left = rank - s.s.found.before;
  auto finish = [&](int first, uint32_t bits) {  // a lane's values, from index first on
    const uint32_t c = __popc(bits), end = wave_prefix(c, Add());
    if (end - c <= left && left < end) {
      for (uint32_t k = left - (end - c); k; --k) bits &= bits - 1;
      a.tokens[m] = first + __builtin_ctz(bits);
      if (a.kept) a.kept[m] = (int32_t)kept;
    }
    return lane_value(end, 63);
  };
  if (seg == 0 || seg == segs - 1) {
    const int first = (seg ? x.head + 8 * x.G : 0) + lane;
    finish(first, first < (seg ? x.V : x.head) && is(x.row[min(first, x.V - 1)]));
    return;
  }
  const int g = 64 * U16 * (seg - 1) + lane;
  uint4 w[U16];
#pragma unroll
  for (int u = 0; u < U16; ++u) w[u] = x.at(g + 64 * u);
#pragma unroll 1
  for (int u = 0; u < U16; ++u) {
    uint32_t bits = 0;
    const uint32_t p[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      bits |= ((uint32_t)is((uint16_t)p[i]) | (uint32_t)is((uint16_t)(p[i] >> 16)) << 1) << 2 * i;
    const uint32_t n = finish(x.head + 8 * (g + 64 * u), g + 64 * u < x.G ? bits : 0u);
    if (left < n) return;
    left -= n;
#pragma unroll
    for (int i = 0; i + 1 < U16; ++i) w[i] = w[i + 1];
  }
}

// False if the row needs the bins of the distance. some: this wave's groups wave + i TT / 64 that
// are not empty.
template <int TT>
__device__ __forceinline__ bool count_row(const TokArgs& a, int m, const Groups<TT>& x, Counts& s,
                                          uint32_t kmax, uint32_t valid, const Row& r,
                                          uint32_t some) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Scale sc{key_value<0>(kmax), 1.4426950408889634 / r.T};
  const double ymin = r.mp > 0.0 ? -log2(r.mp) : INFINITY;
  if (!(fabs(sc.top) < 512.0)) return false;
  if (s.n[2 * ZERO]) {
    const double y = sc.below(-512.f);
    if (y < a.shift + 2 || (r.mp > 0.0 && y <= ymin)) return false;
  }
  // (what is in the bins of +-512 and beyond is not looked for: NaN and no mass)
  auto weight = [&](int bin, double& y) {
    y = sc.below(bf2f((uint16_t)bin_bits(bin)));
    return bin > 0 && bin < 2 * ZERO ? mass_of(y, a.shift) : 0;
  };
  auto number = [&](int bin) { return bin > 0 && bin < 2 * ZERO ? s.n[bin] : 0; };
  // The groups' masses and counts, a wave per group and a bin per lane, two groups at a time:
  // many are empty.
  uint32_t near = 0;
#pragma unroll 1
  while (some) {
    int g[2];
    uint32_t c[2];
    uint64_t mass[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      g[i] = wave + (some ? __builtin_ctz(some) : 31) * (TT / 64);
      c[i] = some ? number(CW * g[i] + lane) : 0;
      some &= some - 1;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      double y;
      mass[i] = c[i] * weight(CW * g[i] + lane, y);
      near += y <= ymin ? c[i] : 0u;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mass[i] = wave_prefix(mass[i], Add());
      c[i] = wave_prefix(c[i], Add());
    }
    if (lane == 63) {
      s.mass[g[0]] = mass[0];
      s.count[g[0]] = c[0];
      if (c[1]) {
        s.mass[g[1]] = mass[1];
        s.count[g[1]] = c[1];
      }
    }
  }
  __syncthreads();
  const uint64_t tm = tid < CG ? s.mass[tid] : 0;
  const uint32_t tc = tid < CG ? s.count[tid] : 0;
  uint64_t pm = tm;
  uint32_t pc = tc;
  block_excl_scan(pm, pc, s.s.s64, s.s.s32);
  if (tid == TT - 1) s.s.found = Found{0, pm + tm, 0, pc + tc, 0};
  if (r.mp > 0.0) near = block_sum<TT / 64>(near, s.s.s32);
  __syncthreads();
  const uint64_t all = s.s.found.own;
  const uint32_t counted = s.s.found.before;

  auto search = [&](uint64_t P, uint32_t K, bool) {
    if (!P && K > counted) return Leaf{0u, K - 1, 1u, all};  // among those without mass
    const uint64_t here = __ballot(!reached(pm, pc, P, K) && reached(pm + tm, pc + tc, P, K));
    if (here) {  // this wave has the group: its bins, one per lane
      const int from = __builtin_ctzll(here);
      const int bin = (64 * wave + from) * CW + lane;
      double y;
      const uint32_t c = number(bin);
      const uint64_t w = weight(bin, y), own = c * w;
      const uint64_t end = wave_prefix(own, Add()) + lane_value(pm, from);
      const uint32_t upto = wave_prefix(c, Add()) + lane_value(pc, from);
      const uint64_t hits = __ballot(reached(end, upto, P, K));
      if (lane == (hits ? __builtin_ctzll(hits) : 63)) {
        Leaf l;
        l.key = (uint32_t)bin;
        l.before = upto - c;
        l.in = min(c, K - l.before);
        if (P && w) l.in = weights_for(P - (end - own), w, l.in);
        l.total = end - own + l.in * w;
        s.s.leaf = l;
      }
    }
    __syncthreads();
    const Leaf l = s.s.leaf;
    __syncthreads();
    return l;
  };
  uint32_t kept;
  const Leaf d = draw_of(r, valid, near, all, kept, search);
  const uint32_t bits = bin_bits((int)d.key);
  pick_bits<TT>(a, x, m, bits | bits << 16, bits ? 0xFFFFFFFFu : 0x7FFF7FFFu, d.in - 1, kept, s);
  return true;
}

template <int TT>
__global__ void __launch_bounds__(TT, 4) sample_tokens_bf16_kernel(TokArgs a) {
  constexpr int CI = (CG + TT / 64 - 1) / (TT / 64);  // groups of a wave
  static_assert(CI < 31, "a bit each");
  extern __shared__ __align__(16) char lds_raw[];
  Counts& s = *reinterpret_cast<Counts*>(lds_raw);
  const int m = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Groups<TT> x(a, m);
  for (int j = tid; j < (int)offsetof(Counts, s) / 16; j += TT)
    reinterpret_cast<uint4*>(s.n)[j] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  x.each([&](int, uint16_t v) { atomicAdd(&s.n[bin_of(v)[0]], 1u); },
         [&](const uint4& v) {
           const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
           for (int i = 0; i < 4; ++i) {
             const u16x2 d = bin_of(w[i]);
             atomicAdd(&s.n[d[0]], 1u);
             atomicAdd(&s.n[d[1]], 1u);
           }
         },
         Never());
  __syncthreads();
  // This wave's groups that are not empty, and the row's first bin that is not.
  uint32_t some = 0, first = 0xFFFFFFFFu;
#pragma unroll
  for (int i = CI - 1; i >= 0; --i) {
    const int g = wave + i * (TT / 64);
    const uint64_t is = __ballot(g < CG && s.n[min(CW * g, CW * (CG - 1)) + lane] != 0);
    some |= (uint32_t)(is != 0) << i;
    if (is) first = CW * g + __builtin_ctzll(is);
  }
  first = ~block_max<TT / 64>(~first, s.s.s32);
  uint32_t kmax = key_of<0>(bf2f((uint16_t)bin_bits((int)first))), valid = (uint32_t)a.V;
  bool tiny = false;
  if (s.n[ZERO]) {  // is it 0?
    uint32_t bad = 0;
    auto look = [&](uint32_t w) {
      bad |= ((w & 0x7FFFu) - 1u < LEAST - 1u) | ((w >> 16 & 0x7FFFu) - 1u < LEAST - 1u);
    };
    x.each([&](int, uint16_t v) { look(v * 0x10001u); },
           [&](const uint4& v) { look(v.x), look(v.y), look(v.z), look(v.w); }, Never());
    tiny = block_max<TT / 64>(bad, s.s.s32) != 0;
  }
  if (tiny || s.n[0] || s.n[2 * ZERO]) maximum<0, TT>(x.row, a.V, kmax, valid, s.s);
  const Row r = row_of(a, m, valid);
  if (simple_row<0, TT>(a, m, kmax, r, s.s)) return;
  if (!tiny && count_row<TT>(a, m, x, s, kmax, valid, r, some)) return;
  __syncthreads();
  general_row<0, TT>(a, m, *reinterpret_cast<General<TT>*>(lds_raw), kmax, valid, r);
}

constexpr int MOST_ROWS = 1 << 22;  // of a launch

template <auto KERN, int TT, int LDS>
int go(const TokArgs& a, hipStream_t st) {
  if (int rc = allow_dynamic_lds<KERN, LDS>()) return rc;
  KERN<<<a.M, TT, LDS, st>>>(a);
  return launch_check("sample_tokens");
}
template <int TT>
int go_type(const TokArgs& a, int dtype, hipStream_t st) {
  constexpr int LDS = (int)sizeof(General<TT>);
  if (dtype == 0)
    return go<sample_tokens_bf16_kernel<TT>, TT, std::max((int)sizeof(Counts), LDS)>(a, st);
  return dtype == 1 ? go<sample_tokens_kernel<1, TT>, TT, LDS>(a, st)
                    : go<sample_tokens_kernel<2, TT>, TT, LDS>(a, st);
}

}  // namespace

extern "C" int grpo_sample_tokens(const void* logits, int dtype, int64_t ld, int M, int V,
                                  const void* draws, int draws_f64, const grpo_sampler_t* sampler,
                                  int64_t* tokens, int32_t* kept, grpo_stream_t stream) {
  if (M < 0 || V < 1 || V > GRPO_SAMPLE_MAX_VOCAB || dtype < 0 || dtype > 2)
    return einval("bad sampling dimensions or dtype");
  if (M == 0) return GRPO_OK;
  if (!logits || !draws || !sampler || !tokens) return einval("null pointer");
  if (M > 1 && ld < V && ld != 0) return einval("rows of logits overlap");
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == 2 ? 4 : 2))
    return einval("logits must be aligned to their type");
  int bits = 0;
  while ((1 << bits) < V) ++bits;
  TokArgs a{logits, ld, M, V, draws, draws_f64, sampler->temperature_rows,
            sampler->top_k_rows, sampler->top_p_rows, sampler->min_p_rows,
            sampler->temperature, sampler->top_p, sampler->min_p, sampler->top_k,
            min(44, 62 - bits), tokens, kept};
  hipStream_t st = as_stream(stream);
  // Fewer waves wait less at the searches' barriers, more read a long row faster: 16 rows of 8000
  // float32 logits 18 us with 512 threads and 24 with 1024, of 40000 29-34 and 33-35, 37 of 50257
  // 38 and 36 (bf16 rows: 1024 from 8000 on).
  const bool small = M > 256 || (dtype != 0 && V <= 49152);
  // (a launch has fewer than 2^32 threads)
  for (int64_t left = M; left > 0; left -= MOST_ROWS) {
    a.M = (int)std::min<int64_t>(left, MOST_ROWS);
    if (int rc = small ? go_type<512>(a, dtype, st) : go_type<1024>(a, dtype, st)) return rc;
    a.logits = static_cast<const char*>(a.logits) + MOST_ROWS * ld * (dtype == 2 ? 4 : 2);
    a.draws = static_cast<const char*>(a.draws) + MOST_ROWS * (draws_f64 ? 8 : 4);
    if (a.temperature) a.temperature += MOST_ROWS;
    if (a.top_k) a.top_k += MOST_ROWS;
    if (a.top_p) a.top_p += MOST_ROWS;
    if (a.min_p) a.min_p += MOST_ROWS;
    a.tokens += MOST_ROWS;
    if (a.kept) a.kept += MOST_ROWS;
  }
  return GRPO_OK;
}

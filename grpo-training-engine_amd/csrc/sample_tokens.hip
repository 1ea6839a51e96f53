// A token from each row of logits with temperature, top-k, top-p and min-p, from given
// uniform numbers (grpo_sample_tokens): the filters of the reference's _sample_tokens
// (src/triton_kernels/paged_kv.py:418-450) in exact arithmetic, without a sort.
//
// Row m: w_v = exp((x_v - max) / T), the row in descending order of x (ties by index). Kept
// is the head of that order with rank < k, then a mass before it below top_p times the mass
// of those k, then w >= min_p; the token is the first kept one at which the running mass
// passes u times the kept mass.
//
//  * Masses are integers, in units of 2^-S of the largest weight, S = 62 - ceil(log2 V), at most
//    44: their sums do not depend on the order in which threads add them, so the token is a
//    function of the inputs alone. Weights are doubles.
//  * "The first place in sorted order where the mass reaches P or the count reaches K" gives the
//    top-k, top-p and min-p cuts and the draw itself. It is found in a histogram of the row: of
//    its values in bf16, else of 4096 distances from the maximum and then, within the one of
//    them that holds the place, of the order-preserving keys until a bin is one value.
//
// A workgroup of 1024 threads per row.
#include <math.h>
#include <stddef.h>

#include <algorithm>

#include "scan.hpp"

using namespace grpo;

namespace {

constexpr int TT = 1024;  // threads
constexpr int SEGS = TT;  // segments of the row in which a tied token is looked for

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

// one(index, value) of the row's values before the first and after the last 16-byte boundary,
// many(index of the first, 16 bytes) of what is between, U loads in flight per thread.
template <int DT, int U, typename One, typename Many>
__device__ __forceinline__ void for_groups(const typename Elem<DT>::type* row, int V, One&& one,
                                           Many&& many) {
  typedef typename Elem<DT>::type E;
  constexpr int N = Elem<DT>::N;
  const int mis = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(E));
  const int head = min(V, mis ? N - mis : 0), G = (V - head) / N, tid = threadIdx.x;
  if (tid < head) one(tid, row[tid]);
  const E* const body = row + head;
  for (int g = tid; g < G; g += U * TT) {
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = *reinterpret_cast<const uint4*>(body + (int64_t)N * min(g + u * TT, G - 1));
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (g + u * TT < G) many(head + N * (g + u * TT), v[u]);
  }
  const int tail = head + N * G + tid;
  if (tail < V) one(tail, row[tail]);
}
// f(index, value as float) of every value.
template <int DT, typename F>
__device__ __forceinline__ void for_row(const typename Elem<DT>::type* row, int V, F&& f) {
  for_groups<DT, 4>(
      row, V, [&](int i, typename Elem<DT>::type x) { f(i, value_of<DT>(x)); },
      [&](int i, const uint4& v) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (DT == 2) {
            f(i + e, __uint_as_float(w[e]));
          } else {
            f(i + 2 * e, value_of<DT>((uint16_t)w[e]));
            f(i + 2 * e + 1, value_of<DT>((uint16_t)(w[e] >> 16)));
          }
        }
      });
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
// A weight in units of 2^-shift; nothing more than shift + 1 doublings below the maximum.
__device__ __forceinline__ uint64_t mass_of(double y, int shift) {
  return y < (double)(shift + 1) ? (uint64_t)rint(exp2_neg(y, shift)) : 0;
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

// Where a search ends: the value, the tokens before it in sorted order, how many of those that
// hold it are needed (1 or more), the mass up to the last of them.
struct Leaf {
  uint32_t key, before, in;
  uint64_t total;
};

// The cuts and the draw, from a search(P, K) for the first place where the mass reaches P (0: no
// such bound) or the count K; `near` tokens pass min_p, `all` is the row's mass.
template <typename Search>
__device__ __forceinline__ Leaf draw_of(const Row& r, uint32_t valid, uint32_t near, uint64_t all,
                                        uint32_t& kept, Search&& search) {
  const uint32_t K = r.mp > 0.0 ? min(r.K, max(near, 1u)) : r.K;
  uint64_t mass = r.K < valid && r.p < 1.0 ? 0 : all;  // of what top_k leaves; then of what is kept
  kept = valid;
  Leaf l;
  // (one place that calls it: the code is large, and once it is there it is there for all three)
#pragma unroll 1
  for (int stage = mass ? 1 : 0; stage < 3; ++stage) {
    const uint64_t P = stage == 0 ? 0 : stage == 2 ? __umul64hi(r.u, mass) + 1
                                  : r.p < 1.0 ? share_of(r.p, mass) : 0;
    if (stage == 1 && !P && K >= valid) continue;
    l = search(P, stage == 0 ? r.K : stage == 1 ? K : kept);
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
  uint64_t s64[TT / 64];
  uint32_t s32[TT / 64];
  Found found;
  Leaf leaf;
  uint32_t n_list, best;
};

// First index of the value with key `key` (all threads get it).
template <int DT>
__device__ __forceinline__ uint32_t first_index(const typename Elem<DT>::type* row, int V,
                                                uint32_t key, Slots& s) {
  if (threadIdx.x == 0) s.best = 0xFFFFFFFFu;
  __syncthreads();
  uint32_t best = 0xFFFFFFFFu;
  for_row<DT>(row, V, [&](int i, float x) {
    if (key_of<DT>(x) == key) best = min(best, (uint32_t)i);
  });
  if (best != 0xFFFFFFFFu) atomicMin(&s.best, best);
  __syncthreads();
  return s.best;
}

// Segments of 2^seg_bits tokens, at most SEGS of them.
__device__ __forceinline__ int seg_bits(int V) { return max(0, 32 - __clz(V - 1) - 10); }
static_assert(SEGS == 1 << 10, "");

// The token of rank `rank` (from 0) by index among those of value `key`, whose numbers per
// segment of 2^seg tokens stand in count: the segment, then the place in it.
template <int DT>
__device__ __forceinline__ void pick(const TokArgs& a, const typename Elem<DT>::type* row, int m,
                                     uint32_t key, uint32_t rank, const uint32_t* count, int seg,
                                     uint32_t kept, Slots& s) {
  const int tid = threadIdx.x, V = a.V;
  uint64_t unused = 0;
  const uint32_t mine = count[tid];
  uint32_t upto = mine;
  block_excl_scan(unused, upto, s.s64, s.s32);
  if (upto <= rank && rank < upto + mine) {
    s.found.bin = tid;
    s.found.before = upto;
  }
  __syncthreads();
  if (tid >= 64) return;
  const int i0 = (int)s.found.bin << seg, i1 = min(V, i0 + (1 << seg));
  uint32_t left = rank - s.found.before;
  for (int i = i0; i < i1; i += 64) {
    const int at = i + tid;
    const bool hit = at < i1 && key_of<DT>(value_of<DT>(row[min(at, V - 1)])) == key;
    const uint64_t hits = __ballot(hit);
    const uint32_t n = __popcll(hits);
    if (left < n) {
      if (hit && (uint32_t)__popcll(hits & ((1ull << tid) - 1)) == left) {
        a.tokens[m] = at;
        if (a.kept) a.kept[m] = (int32_t)kept;
      }
      return;
    }
    left -= n;
  }
}

// ------------------------------------------------- bins of the distance --
// 64 bins per doubling below the maximum. A token adds one 64-bit number to its bin: 1 to the
// count in the upper bits, and (1 - 2^-(f / 64)) 2^UNIT to a sum in the lower ones, f its place in
// the bin. A bin's mass is 2^-(bin / 64) (count - sum): one LDS atomic and 5 FMAs per token
// instead of two and an exponential. Within a bin the tokens' weights are relative to the bin's
// first, and P is a share of the bin's mass.
constexpr int NB = 4096;
constexpr int PER = NB / TT;   // bins of a thread
constexpr int NK = TT;         // bins of keys
constexpr int KEY_BITS = 10;
constexpr int LIST = 4096;     // tokens of one bin that LDS holds
constexpr double A64 = 0.010830424696249145;  // ln(2) / 64

struct General {
  unsigned long long bins[NB];
  unsigned long long kmass[NK];
  uint32_t kcnt[NK];
  uint32_t lkey[LIST];
  uint32_t lidx[LIST];
  Slots s;
};

__device__ __forceinline__ double bin_place(double y) { return fmin(y * 64.0, (double)(NB - 1)); }

// Smallest key in [1, kmax] whose bin is at most j: 64 candidates at a time.
template <int DT>
__device__ __forceinline__ uint32_t first_key(const Scale& sc, uint32_t kmax, int j) {
  uint32_t lo = 1, hi = kmax;  // hi holds
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

template <int DT>
__device__ __forceinline__ void general_row(const TokArgs& a, int m, General& s, uint32_t kmax,
                                            uint32_t valid, const Row& r) {
  typedef typename Elem<DT>::type E;
  const int tid = threadIdx.x, V = a.V;
  const E* const row = static_cast<const E*>(a.logits) + (int64_t)m * a.ld;
  const Scale sc{key_value<DT>(kmax), 1.4426950408889634 / r.T};
  const double ymin = r.mp > 0.0 ? -log2(r.mp) : INFINITY;
  // units of a place's sum: the sum of V of them, below V A64, stays in the lower bits
  const int cbits = a.V < 1 << 18 ? 18 : 21, unit = 70 - 2 * cbits;
  const int sbits = 64 - cbits;
  for (int j = tid; j < NB; j += TT) s.bins[j] = 0;
  if (tid == 0) s.s.n_list = 0;
  __syncthreads();
  uint32_t near = 0;  // tokens that min_p leaves
  {
    const double sl = ldexp(1.0, unit), k1 = A64 * sl, k2 = -A64 * A64 / 2 * sl,
                 k3 = A64 * A64 * A64 / 6 * sl, k4 = -A64 * A64 * A64 * A64 / 24 * sl,
                 k5 = A64 * A64 * A64 * A64 * A64 / 120 * sl;
    for_row<DT>(row, V, [&](int, float x) {
      if (!(x > -INFINITY)) return;
      const double y = sc.below(x);
      near += y <= ymin ? 1u : 0u;
      const double z = bin_place(y);
      const int b = (int)z;
      const double f = z - b;
      // (the double's last place is 1 after 2^52 is added)
      const double q = fma(fma(fma(fma(fma(k5, f, k4), f, k3), f, k2), f, k1), f, 4503599627370496.0);
      const uint64_t lo = (uint64_t)__double_as_longlong(q) & ((1ull << 52) - 1);
      atomicAdd(&s.bins[b], (unsigned long long)(lo + (1ull << sbits)));
    });
  }
  near = block_sum<TT / 64>(near, s.s.s32);
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

  int listed = -1, last = -1;  // bins: whose tokens stand in the list, that held the last place
  auto search = [&](uint64_t P, uint32_t K) {
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
    uint32_t lo = first_key<DT>(sc, kmax, bin);
    uint32_t hi = bin ? first_key<DT>(sc, kmax, bin - 1) - 1 : kmax;
    const bool list = top.group <= LIST;
    if (list && listed != bin) {
      if (tid == 0) s.s.n_list = 0;
      __syncthreads();
      for_row<DT>(row, V, [&](int i, float x) {
        const uint32_t k = key_of<DT>(x);
        if (k < lo || k > hi) return;
        const uint32_t at = atomicAdd(&s.s.n_list, 1u);
        if (at >= LIST) return;  // (never: the bin holds as many)
        s.lkey[at] = k;
        s.lidx[at] = i;
      });
      listed = bin;
    }
    __syncthreads();
    const uint32_t n = min(s.s.n_list, (uint32_t)LIST);
    // weights relative to the bin's start: 2^44 of it at most
    auto rel = [&](uint32_t k) {
      return (uint64_t)rint(exp2_neg(fmax(sc.below(key_value<DT>(k)) - bin * (1.0 / 64), 0.0), a.shift));
    };
    uint64_t Q = 0, mb = 0, sum = 0;  // P in those, before the range, of the whole bin
    uint32_t cb = top.before, group = top.group;
    bool first = true;
    while (lo < hi) {
      const int sh = max(0, 32 - __clz(hi - lo) - KEY_BITS);
      for (int j = tid; j < NK; j += TT) {
        s.kmass[j] = 0;
        s.kcnt[j] = 0;
      }
      __syncthreads();
      auto add = [&](uint32_t k) {
        if (k < lo || k > hi) return;
        atomicAdd(&s.kmass[(hi - k) >> sh], (unsigned long long)rel(k));
        atomicAdd(&s.kcnt[(hi - k) >> sh], 1u);
      };
      if (list) {
        for (uint32_t i = tid; i < n; i += TT) add(s.lkey[i]);
      } else {
        for_row<DT>(row, V, [&](int, float x) { add(key_of<DT>(x)); });
      }
      __syncthreads();
      const uint64_t mt = s.kmass[tid];
      const uint32_t ct = s.kcnt[tid];
      uint64_t before = mt;
      uint32_t upto = ct;
      block_excl_scan(before, upto, s.s.s64, s.s.s32);
      if (first) {
        sum = block_sum<TT / 64>(mt, s.s.s64);
        // (a bin whose tokens have no mass of their own: the last one)
        Q = P ? (top.own ? (uint64_t)ceil((double)(P - top.mass) / (double)top.own * (double)sum)
                         : sum) : 0;
        Q = P > top.mass + top.own ? 0 : min(max(Q, (uint64_t)(P ? 1 : 0)), sum);
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
    }
    const uint64_t w = rel(hi);
    if (first) {  // the bin is one value
      sum = w * group;
      Q = P && P <= top.mass + top.own && top.own
              ? max((uint64_t)1, (uint64_t)ceil((double)(P - top.mass) / (double)top.own * (double)sum))
              : 0;
    }
    Leaf l;
    l.key = hi;
    l.before = cb;
    l.in = min(group, K - cb);
    if (Q) {
      const uint64_t need = (Q - mb + w - 1) / w;  // (w >= 2^43 / 2^(1/64))
      if (need < l.in) l.in = (uint32_t)need;
    }
    l.in = max(l.in, 1u);
    const uint64_t end = mb + l.in * w;
    l.total = top.mass + (end >= sum ? top.own
                                     : (uint64_t)rint((double)end / (double)sum * (double)top.own));
    if (l.total == 0) l.total = 1;
    return l;
  };

  uint32_t kept;
  const Leaf d = draw_of(r, valid, near, all, kept, search);
  const int seg = seg_bits(V);
  s.kcnt[tid] = 0;
  __syncthreads();
  if (listed == last) {
    for (uint32_t i = tid; i < min(s.s.n_list, (uint32_t)LIST); i += TT)
      if (s.lkey[i] == d.key) atomicAdd(&s.kcnt[s.lidx[i] >> seg], 1u);
  } else {
    for_row<DT>(row, V, [&](int i, float x) {
      if (key_of<DT>(x) == d.key) atomicAdd(&s.kcnt[i >> seg], 1u);
    });
  }
  __syncthreads();
  pick<DT>(a, row, m, d.key, d.in - 1, s.kcnt, seg, kept, s.s);
}

template <int DT>
__device__ __forceinline__ void maximum(const typename Elem<DT>::type* row, int V, uint32_t& kmax,
                                        uint32_t& valid, Slots& s) {
  kmax = valid = 0;
  for_row<DT>(row, V, [&](int, float x) {
    const uint32_t k = key_of<DT>(x);
    kmax = max(kmax, k);
    valid += k ? 1u : 0u;
  });
  kmax = block_max<TT / 64>(kmax, s.s32);
  valid = block_sum<TT / 64>(valid, s.s32);
}

// Rows with nothing to draw, or whose maximum is taken; true if done.
template <int DT>
__device__ __forceinline__ bool simple_row(const TokArgs& a, int m, uint32_t kmax, const Row& r,
                                           Slots& s) {
  typedef typename Elem<DT>::type E;
  if (kmax && !r.greedy) return false;
  int64_t token = -1;
  if (kmax)
    token = first_index<DT>(static_cast<const E*>(a.logits) + (int64_t)m * a.ld, a.V, kmax, s);
  if (threadIdx.x == 0) {
    a.tokens[m] = token;
    if (a.kept) a.kept[m] = kmax ? 1 : 0;
  }
  return true;
}

// ------------------------------------------------------- bf16: its values --
// A bf16 row has few distinct values: their counts, one 32-bit LDS atomic per token, and a
// weight per value. The bins are fixed, the values of magnitude below 512 in descending order,
// so that one pass over the row makes the counts and finds the maximum. A row with a larger
// maximum, or with mass at -512 and below (an extreme temperature), takes the bins of the distance.
// (The row in registers instead of its second reading: 8 / 512 rows of 151936 39 / 155 us against
// 35 / 100, in code without loops that runs at the rate of its instruction fetches.)
constexpr int CW = 64;              // bins of a group: one per lane
constexpr int CG = 544;             // groups: one per thread
constexpr int CB = CW * CG;
constexpr int CI = CG / (TT / 64);  // groups of a wave
constexpr int TOP = CB / 2;         // the bin of t is TOP - 1 - t
static_assert(CG % (TT / 64) == 0 && CG <= TT, "groups split evenly");
static_assert(TOP == 0x4400, "the bits of 512");
constexpr int SEG_PER = 3;          // segments of a thread in the search for a token
typedef int16_t s16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

struct Counts {
  uint32_t n[CB + 32];  // n[CB]: of what has no bin
  uint64_t mass[CG];    // of the groups
  uint32_t count[CG];   // (all of these are zero at first)
  Slots s;
};

// The value's bits as a 16-bit integer in the order of the values: +0 -> 0, -0 -> -1; +inf,
// and what is a NaN above it; -inf, and what is a NaN below it.
constexpr int T_INF = 0x7F80, T_NINF = 0x7F - 0x8000;
__device__ __forceinline__ s16x2 order_of(uint32_t pair) {
  const s16x2 x = __builtin_bit_cast(s16x2, pair);
  return x ^ ((x >> 15) & (int16_t)0x7FFF);
}
__device__ __forceinline__ float ordered_value(int t) {
  return bf2f((uint16_t)(t < 0 ? t ^ 0x7FFF : t));
}

// Where the row's 16-byte groups begin, and how many they are.
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
    return *reinterpret_cast<const uint4*>(row + head + 8 * (int64_t)g);
  }
  // one(0 or 1, index, value) of the values before and after the groups, many(g, group)
  template <typename One, typename Many>
  __device__ __forceinline__ void each(One&& one, Many&& many) const {
    constexpr int U = 8;
    const int tid = threadIdx.x, tail = head + 8 * G + tid;
    if (tid < head) one(0, tid, row[tid]);
#pragma unroll 1
    for (int g = tid; g < G; g += U * TT) {
      uint4 w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = at(min(g + u * TT, G - 1));
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (g + u * TT < G) many(g + u * TT, w[u]);
    }
    if (tail < V) one(1, tail, row[tail]);
  }
};

// The token of rank `rank` among those whose bits are want (two of them, compared in mask),
// counted per wave's groups; all threads get it.
__device__ __forceinline__ void pick_bits(const TokArgs& a, const Groups& x, int m, uint32_t want,
                                          uint32_t mask, uint32_t rank, uint32_t kept, Counts& s) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int segs = 2 + (x.G + 63) / 64;  // before the groups, 64 groups each, after them
  for (int j = tid; j < SEG_PER * TT; j += TT) s.n[j] = 0;
  __syncthreads();
  auto matches = [&](const uint4& w) {
    const uint32_t p[4] = {w.x, w.y, w.z, w.w};
    const u16x2 one = (uint16_t)1;
    u16x2 not_it = (uint16_t)0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      not_it += __builtin_elementwise_min(__builtin_bit_cast(u16x2, (p[i] ^ want) & mask), one);
    return 8u - not_it[0] - not_it[1];
  };
  auto is = [&](uint16_t v) { return ((v ^ want) & mask & 0xFFFFu) == 0; };
  x.each(
      [&](int end, int, uint16_t v) {
        if (is(v)) atomicAdd(&s.n[end ? segs - 1 : 0], 1u);
      },
      [&](int g, const uint4& w) {
        const uint32_t c = matches(w);
        if (c) atomicAdd(&s.n[1 + g / 64], c);
      });
  __syncthreads();
  uint32_t c[SEG_PER], mine = 0, upto;
#pragma unroll
  for (int j = 0; j < SEG_PER; ++j) mine += c[j] = s.n[SEG_PER * tid + j];
  upto = mine;
  uint64_t unused = 0;
  block_excl_scan(unused, upto, s.s.s64, s.s.s32);
  if (upto <= rank && rank < upto + mine) {
#pragma unroll
    for (int j = 0; j < SEG_PER; ++j) {
      if (upto <= rank && rank < upto + c[j]) s.s.found = Found{0, 0, (uint32_t)(SEG_PER * tid + j), upto, 0};
      upto += c[j];
    }
  }
  __syncthreads();
  if (tid >= 64) return;
  const int seg = (int)s.s.found.bin;
  const uint32_t left = rank - s.s.found.before;
  // a lane's values: a group's eight, or one of an end
  const int g = 64 * (seg - 1) + lane;
  const bool ends = seg == 0 || seg == segs - 1;
  const int first = ends ? (seg ? x.head + 8 * x.G : 0) + lane : x.head + 8 * g;
  const int count = ends ? (first < (seg ? x.V : x.head) ? 1 : 0) : (g < x.G ? 8 : 0);
  uint32_t bits = 0;
  for (int i = 0; i < count; ++i) bits |= (uint32_t)is(x.row[first + i]) << i;
  const uint32_t before = wave_prefix((uint32_t)__popc(bits), Add()) - __popc(bits);
  if (before <= left && left < before + __popc(bits)) {
    for (uint32_t k = left - before; k; --k) bits &= bits - 1;
    a.tokens[m] = first + __builtin_ctz(bits);
    if (a.kept) a.kept[m] = (int32_t)kept;
  }
}

// False if the row needs the bins of the distance.
__device__ __forceinline__ bool count_row(const TokArgs& a, int m, const Groups& x, Counts& s,
                                          uint32_t kmax, uint32_t valid, const Row& r) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Scale sc{key_value<0>(kmax), 1.4426950408889634 / r.T};
  const double ymin = r.mp > 0.0 ? -log2(r.mp) : INFINITY;
  if (!(fabs(sc.top) < 512.0)) return false;
  if (s.n[CB]) {
    const double y = sc.below(-512.f);
    if (y < a.shift + 2 || (r.mp > 0.0 && y <= ymin)) return false;
  }
  auto distance = [&](int bin) { return sc.below(ordered_value(TOP - 1 - bin)); };
  // The groups' masses and counts, a wave per group and a bin per lane: most groups are empty,
  // and the others stand side by side.
  uint32_t near = 0;
  {
    uint64_t some = 0;  // of this wave's groups
#pragma unroll
    for (int i = 0; i < CI; ++i)
      some |= (uint64_t)(__ballot(s.n[CW * (wave + i * (TT / 64)) + lane] != 0) != 0) << i;
#pragma unroll 1
    for (; some; some &= some - 1) {
      const int g = wave + __builtin_ctzll(some) * (TT / 64);
      const uint32_t c = s.n[CW * g + lane];
      const double y = distance(CW * g + lane);
      const uint64_t mass = wave_prefix(c * mass_of(y, a.shift), Add());
      const uint32_t count = wave_prefix(c, Add());
      near += y <= ymin ? c : 0u;
      if (lane == 63) {
        s.mass[g] = mass;
        s.count[g] = count;
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
  __syncthreads();

  int found = 0;  // bin of the last search
  auto search = [&](uint64_t P, uint32_t K) {
    if (!P && K > counted) return Leaf{0u, K - 1, 1u, all};  // among those without mass
    if (!reached(pm, pc, P, K) && reached(pm + tm, pc + tc, P, K))
      s.s.found = Found{pm, 0, (uint32_t)tid, pc, 0};
    __syncthreads();
    const Found f = s.s.found;
    const int bin = (int)f.bin * CW + lane;
    const uint32_t c = s.n[bin];
    const uint64_t w = mass_of(distance(bin), a.shift), own = c * w;
    const uint64_t end = wave_prefix(own, Add()) + f.mass;
    const uint32_t upto = wave_prefix(c, Add()) + f.before;
    const uint64_t hits = __ballot(reached(end, upto, P, K));
    const int at = hits ? __builtin_ctzll(hits) : 63;
    found = (int)f.bin * CW + at;
    const uint64_t own_at = lane_value(own, at), w_at = lane_value(w, at);
    const uint64_t before = lane_value(end, at) - own_at;
    const uint32_t c_at = lane_value(c, at);
    Leaf l;
    l.before = lane_value(upto, at) - c_at;
    l.in = min(c_at, K - l.before);
    if (P && w_at) l.in = (uint32_t)min((uint64_t)l.in, (P - before + w_at - 1) / w_at);
    l.key = 0;
    l.total = before + l.in * w_at;
    __syncthreads();  // found has been read
    return l;
  };
  uint32_t kept;
  const Leaf d = draw_of(r, valid, near, all, kept, search);
  const int t = TOP - 1 - found;  // (-0 stands with +0)
  const uint32_t bits = (uint32_t)(t < 0 ? t ^ 0x7FFF : t) & 0xFFFFu;
  pick_bits(a, x, m, bits | bits << 16, bits ? 0xFFFFFFFFu : 0x7FFF7FFFu, d.in - 1, kept, s);
  return true;
}

__global__ void __launch_bounds__(TT) sample_tokens_bf16_kernel(TokArgs a) {
  extern __shared__ __align__(16) char lds_raw[];
  Counts& s = *reinterpret_cast<Counts*>(lds_raw);
  const int m = blockIdx.x;
  const Groups x(a, m);
  static_assert(offsetof(Counts, s) % 16 == 0, "cleared 16 bytes at a time");
  for (int j = threadIdx.x; j < (int)offsetof(Counts, s) / 16; j += TT)
    reinterpret_cast<uint4*>(s.n)[j] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  s16x2 hi = (int16_t)-0x8000, lo = (int16_t)0x7FFF;
  const u16x2 top = (uint16_t)(TOP - 1), none = (uint16_t)CB;
  auto pair = [&](uint32_t w) {
    const s16x2 t = order_of(w);
    hi = __builtin_elementwise_max(hi, t);
    lo = __builtin_elementwise_min(lo, t);
    return __builtin_elementwise_min(top - __builtin_bit_cast(u16x2, t), none);
  };
  x.each([&](int, int, uint16_t v) { atomicAdd(&s.n[pair(v * 0x10001u)[0]], 1u); },
         [&](int, const uint4& v) {
           const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
           for (int i = 0; i < 4; ++i) {
             const u16x2 d = pair(w[i]);
             atomicAdd(&s.n[d[0]], 1u);
             atomicAdd(&s.n[d[1]], 1u);
           }
         });
  const int most = max((int)hi[0], (int)hi[1]), least = min((int)lo[0], (int)lo[1]);
  const int tmax = (int)block_max<TT / 64>((uint32_t)(most + 0x8000), s.s.s32) - 0x8000;
  const int tmin = 0x8000 - (int)block_max<TT / 64>((uint32_t)(0x8000 - least), s.s.s32);
  uint32_t kmax = key_of<0>(ordered_value(tmax)), valid = (uint32_t)a.V;
  if (tmax > T_INF || tmin <= T_NINF)  // NaN or -inf among them
    maximum<0>(x.row, a.V, kmax, valid, s.s);
  if (threadIdx.x == 0) {  // -0 with +0
    s.n[TOP - 1] += s.n[TOP];
    s.n[TOP] = 0;
  }
  __syncthreads();
  const Row r = row_of(a, m, valid);
  if (simple_row<0>(a, m, kmax, r, s.s)) return;
  if (count_row(a, m, x, s, kmax, valid, r)) return;
  __syncthreads();
  general_row<0>(a, m, *reinterpret_cast<General*>(lds_raw), kmax, valid, r);
}

template <int DT>
__global__ void __launch_bounds__(TT) sample_tokens_kernel(TokArgs a) {
  typedef typename Elem<DT>::type E;
  extern __shared__ __align__(16) char lds_raw[];
  General& s = *reinterpret_cast<General*>(lds_raw);
  const int m = blockIdx.x;
  uint32_t kmax, valid;
  maximum<DT>(static_cast<const E*>(a.logits) + (int64_t)m * a.ld, a.V, kmax, valid, s.s);
  const Row r = row_of(a, m, valid);
  if (simple_row<DT>(a, m, kmax, r, s.s)) return;
  general_row<DT>(a, m, s, kmax, valid, r);
}

template <auto KERN, int LDS>
int go(const TokArgs& a, hipStream_t st) {
  if (int rc = allow_dynamic_lds<KERN, LDS>()) return rc;
  KERN<<<a.M, TT, LDS, st>>>(a);
  return launch_check("sample_tokens");
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
  const TokArgs a{logits, ld, M, V, draws, draws_f64, sampler->temperature_rows,
                  sampler->top_k_rows, sampler->top_p_rows, sampler->min_p_rows,
                  sampler->temperature, sampler->top_p, sampler->min_p, sampler->top_k,
                  min(44, 62 - bits), tokens, kept};
  hipStream_t st = as_stream(stream);
  constexpr int LDS = (int)sizeof(General);
  constexpr int LDS16 = (int)std::max(sizeof(Counts), sizeof(General));
  if (dtype == 0) return go<sample_tokens_bf16_kernel, LDS16>(a, st);
  return dtype == 1 ? go<sample_tokens_kernel<1>, LDS>(a, st)
                    : go<sample_tokens_kernel<2>, LDS>(a, st);
}

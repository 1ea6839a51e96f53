// A token from each row of logits with temperature, top-k, top-p and min-p, from given
// uniform numbers (grpo_sample_tokens): the filters of the reference's _sample_tokens
// (src/triton_kernels/paged_kv.py:418-450) in exact arithmetic, without a sort.
//
// Row m: w_v = exp((x_v - max) / T), the row in descending order of x (ties by index). Kept
// is the head of that order with rank < k, then a mass before it below top_p times the mass
// of those k, then w >= min_p; the token is the first kept one at which the running mass
// passes u times the kept mass.
//
//  * Masses are integers: w in units of 2^-S, S = 62 - ceil(log2 V), at most 44. Their sums do
//    not depend on the order in which threads add them, so the token is a function of the
//    inputs alone. A weight is a double (degree-11 Taylor polynomial of 2^f on [-1/2, 1/2],
//    below 1e-14 relative) rounded once to those units; what is more than 45 doublings below
//    the maximum has no mass.
//  * "The first place in sorted order where the mass reaches P or the count reaches K" is
//    found by descending through ranges of order-preserving keys: 4096 bins of the distance
//    from the maximum, then bins of the keys within one bin until a bin is one value. That
//    one search gives the top-k, top-p and min-p cuts and the draw itself.
#include <math.h>

#include "scan.hpp"

using namespace grpo;

namespace {

constexpr int TT = 1024;           // threads
constexpr int NB = 4096;           // bins of the distance from the maximum
constexpr double WINDOW = 48.0;    // doublings that they cover (the last takes the rest)
constexpr int NK = 2048;           // bins of keys
constexpr int KEY_BITS = 11;
constexpr int LIST = 8192;         // values of one bin that LDS holds
constexpr int SEGS = 2048;         // segments of the row in which a tied token is looked for

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
__device__ __forceinline__ float value_of(uint32_t bits) {
  if constexpr (DT == 0) return bf2f((uint16_t)bits);
  if constexpr (DT == 1) return h2f((uint16_t)bits);
  return __uint_as_float(bits);
}

// f(index, value) of every value of the row; 16-byte loads from the first boundary on.
template <int DT, typename F>
__device__ __forceinline__ void for_row(const typename Elem<DT>::type* row, int V, F&& f) {
  typedef typename Elem<DT>::type E;
  constexpr int N = Elem<DT>::N, U = 4;
  const int mis = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(E));
  const int head = min(V, mis ? N - mis : 0), G = (V - head) / N, tid = threadIdx.x;
  auto scalar = [&](int i) {
    if constexpr (DT == 2)
      f(i, row[i]);
    else
      f(i, value_of<DT>(row[i]));
  };
  if (tid < head) scalar(tid);
  const E* const body = row + head;
  for (int g = tid; g < G; g += U * TT) {
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = *reinterpret_cast<const uint4*>(body + (int64_t)N * min(g + u * TT, G - 1));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (g + u * TT >= G) break;
      const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
      const int at = head + N * (g + u * TT);
#pragma unroll
      for (int e = 0; e < N; ++e)
        f(at + e, value_of<DT>(DT == 2 ? w[e & 3] : ((e & 1) ? w[(e >> 1) & 3] >> 16
                                                             : w[(e >> 1) & 3] & 0xFFFFu)));
    }
  }
  const int tail = head + N * G + tid;
  if (tail < V) scalar(tail);
}

// Distance from the maximum in doublings (0 at the maximum itself, infinite ones included;
// infinite for what has no mass).
struct Scale {
  float top;
  double c;  // log2(e) / T
  __device__ __forceinline__ double below(float x) const {
    const double y = ((double)top - (double)x) * c;
    return x == top ? 0.0 : (y >= 0.0 ? y : (double)INFINITY);
  }
};
__device__ __forceinline__ int bin_of(double y) {
  return (int)fmin(y * (NB / WINDOW), (double)(NB - 1));
}

// round(2^(S - y)): the double's last place is 1 after 2^52 is added.
__device__ __forceinline__ uint64_t mass_of(double y, int shift) {
  if (!(y < (double)(shift + 1))) return 0;
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
  const double r = ldexp(p, shift - (int)n) + 4503599627370496.0;
  return (uint64_t)__double_as_longlong(r) & ((1ull << 52) - 1);
}

struct Lds {
  unsigned long long mass[NB];
  unsigned long long kmass[NK];
  uint32_t cnt[NB];
  uint32_t kcnt[NK];
  uint32_t lkey[LIST];
  uint32_t lidx[LIST];
  uint64_t s64[TT / 64];
  uint32_t s32[TT / 64];
  uint64_t f_mass;  // of find()
  uint32_t f_bin, f_cnt;
  uint32_t n_list, best;
};

// Where a search ends: the value (key), what stands before it in sorted order, how many tokens
// hold it and how many of those are needed.
struct Leaf {
  uint32_t key;
  uint64_t mass;
  uint32_t before, group, in;
  uint64_t w;
  int bin;
  __device__ uint32_t count() const { return before + in; }
  __device__ uint64_t total() const { return mass + in * w; }
};

// The first of N bins at whose end the mass reaches P (0: no such bound) or the count K.
template <int N>
__device__ __forceinline__ void find(Lds& s, const unsigned long long* mass, const uint32_t* cnt,
                                     uint64_t mb, uint32_t cb, uint64_t P, uint32_t K) {
  constexpr int PER = N / TT;
  const int b0 = threadIdx.x * PER;
  uint64_t m = 0;
  uint32_t c = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    m += mass ? mass[b0 + j] : 0;
    c += cnt[b0 + j];
  }
  uint64_t pm = m;
  uint32_t pc = c;
  if (threadIdx.x == 0) {  // (a bound always lies within the bins)
    s.f_bin = N - 1;
    s.f_mass = mb;
    s.f_cnt = cb;
  }
  block_excl_scan(pm, pc, s.s64, s.s32);
  pm += mb;
  pc += cb;
  auto reached = [&](uint64_t a, uint32_t b) { return (P && a >= P) || b >= K; };
  if (!reached(pm, pc) && reached(pm + m, pc + c)) {
    for (int j = 0; j < PER; ++j) {
      const uint64_t mj = mass ? mass[b0 + j] : 0;
      const uint32_t cj = cnt[b0 + j];
      if (reached(pm + mj, pc + cj)) {
        s.f_bin = b0 + j;
        s.f_mass = pm;
        s.f_cnt = pc;
        break;
      }
      pm += mj;
      pc += cj;
    }
  }
  __syncthreads();
}

// Smallest key in [1, kmax] whose bin is at most j: 64 candidates at a time.
template <int DT>
__device__ __forceinline__ uint32_t first_key(const Scale& sc, uint32_t kmax, int j) {
  uint32_t lo = 1, hi = kmax;  // hi holds
  while (lo < hi) {
    const uint32_t step = (hi - lo) / 64 + 1, lane = threadIdx.x & 63;
    const uint32_t c = (uint32_t)min((uint64_t)lo + (uint64_t)lane * step, (uint64_t)hi);
    const uint64_t is = __ballot(bin_of(sc.below(key_value<DT>(c))) <= j);
    const uint32_t f = is ? __builtin_ctzll(is) : 64;
    const uint32_t at = lo;
    if (f < 64) hi = (uint32_t)min((uint64_t)at + (uint64_t)f * step, (uint64_t)hi);
    lo = f ? at + (f - 1) * step + 1 : at;
    if (f == 0) hi = at;
  }
  return hi;
}

template <int DT>
__global__ void __launch_bounds__(TT) sample_tokens_kernel(TokArgs a) {
  typedef typename Elem<DT>::type E;
  extern __shared__ __align__(16) char lds_raw[];
  Lds& s = *reinterpret_cast<Lds*>(lds_raw);
  const int tid = threadIdx.x, m = blockIdx.x, V = a.V;
  const E* const row = static_cast<const E*>(a.logits) + (int64_t)m * a.ld;

  uint32_t kmax = 0, valid = 0;
  for_row<DT>(row, V, [&](int, float x) {
    const uint32_t k = key_of<DT>(x);
    kmax = max(kmax, k);
    valid += k ? 1u : 0u;
  });
  kmax = block_max<TT / 64>(kmax, s.s32);
  valid = block_sum<TT / 64>(valid, s.s32);
  if (kmax == 0) {  // nothing to draw
    if (tid == 0) {
      a.tokens[m] = -1;
      if (a.kept) a.kept[m] = 0;
    }
    return;
  }
  const double T = a.temperature ? (double)a.temperature[m] : a.t;
  const int64_t topk = a.top_k ? (int64_t)a.top_k[m] : a.k;
  const double p = a.top_p ? (double)a.top_p[m] : a.p;
  const double mp = a.min_p ? (double)a.min_p[m] : a.mp;
  uint32_t K = topk > 0 && topk < (int64_t)valid ? (uint32_t)topk : valid;
  if (!(T > 0.0) || p <= 0.0 || mp > 1.0) K = 1;
  if (K == 1) {  // the lowest index of the maximum
    if (tid == 0) s.best = 0xFFFFFFFFu;
    __syncthreads();
    uint32_t best = 0xFFFFFFFFu;
    for_row<DT>(row, V, [&](int i, float x) {
      if (key_of<DT>(x) == kmax) best = min(best, (uint32_t)i);
    });
    if (best != 0xFFFFFFFFu) atomicMin(&s.best, best);
    __syncthreads();
    if (tid == 0) {
      a.tokens[m] = s.best;
      if (a.kept) a.kept[m] = 1;
    }
    return;
  }

  const Scale sc{key_value<DT>(kmax), 1.4426950408889634 / T};
  const double ymin = mp > 0.0 ? -log2(mp) : INFINITY;
  for (int j = tid; j < NB; j += TT) {
    s.mass[j] = 0;
    s.cnt[j] = 0;
  }
  if (tid == 0) s.n_list = 0;
  __syncthreads();
  uint32_t near = 0;  // tokens that min_p leaves
  uint64_t all = 0;
  for_row<DT>(row, V, [&](int, float x) {
    if (!key_of<DT>(x)) return;
    const double y = sc.below(x);
    const int b = bin_of(y);
    const uint64_t w = mass_of(y, a.shift);
    atomicAdd(&s.mass[b], (unsigned long long)w);
    atomicAdd(&s.cnt[b], 1u);
    all += w;
    near += y <= ymin ? 1u : 0u;
  });
  near = block_sum<TT / 64>(near, s.s32);
  all = block_sum<TT / 64>(all, s.s64);

  int listed = -1;  // the bin whose tokens stand in the list
  auto descend = [&](uint64_t P, uint32_t bound) {
    find<NB>(s, s.mass, s.cnt, 0, 0, P, bound);
    Leaf r;
    const int bin = r.bin = s.f_bin;
    r.mass = s.f_mass;
    r.before = s.f_cnt;
    r.group = s.cnt[bin];
    uint32_t lo = first_key<DT>(sc, kmax, bin);
    uint32_t hi = bin ? first_key<DT>(sc, kmax, bin - 1) - 1 : kmax;
    const bool list = r.group <= LIST;
    __syncthreads();
    if (list && listed != bin) {
      if (tid == 0) s.n_list = 0;
      __syncthreads();
      for_row<DT>(row, V, [&](int i, float x) {
        const uint32_t k = key_of<DT>(x);
        if (k < lo || k > hi) return;
        const uint32_t at = atomicAdd(&s.n_list, 1u);
        if (at >= LIST) return;  // (never: the bin holds as many)
        s.lkey[at] = k;
        s.lidx[at] = i;
      });
      listed = bin;
      __syncthreads();
    }
    while (lo < hi) {
      const int sh = max(0, 32 - __clz(hi - lo) - KEY_BITS);
      for (int j = tid; j < NK; j += TT) {
        s.kmass[j] = 0;
        s.kcnt[j] = 0;
      }
      __syncthreads();
      auto add = [&](uint32_t k) {
        if (k < lo || k > hi) return;
        const uint32_t q = (hi - k) >> sh;
        atomicAdd(&s.kmass[q], (unsigned long long)mass_of(sc.below(key_value<DT>(k)), a.shift));
        atomicAdd(&s.kcnt[q], 1u);
      };
      if (list) {
        for (uint32_t i = tid; i < min(s.n_list, (uint32_t)LIST); i += TT) add(s.lkey[i]);
      } else {
        for_row<DT>(row, V, [&](int, float x) { add(key_of<DT>(x)); });
      }
      __syncthreads();
      find<NK>(s, s.kmass, s.kcnt, r.mass, r.before, P, bound);
      const uint32_t q = min(s.f_bin, (hi - lo) >> sh);
      r.mass = s.f_mass;
      r.before = s.f_cnt;
      r.group = s.kcnt[q];
      hi -= q << sh;
      const uint32_t width = (1u << sh) - 1;
      if (hi - lo > width) lo = hi - width;
      __syncthreads();
    }
    r.key = hi;
    r.w = mass_of(sc.below(key_value<DT>(hi)), a.shift);
    r.in = min(r.group, bound - r.before);
    if (P && r.w) {
      const uint64_t need = (P - r.mass + r.w - 1) / r.w;
      if (need < r.in) r.in = (uint32_t)need;
    }
    return r;
  };

  uint64_t P = 0;
  if (p < 1.0) {
    const uint64_t most = K < valid ? descend(0, K).total() : all;
    const uint64_t pf = (uint64_t)(p * 18446744073709551616.0);
    P = __umul64hi(pf, most) + (pf * most ? 1 : 0);
    if (P == 0) P = 1;
  }
  K = min(K, max(near, 1u));
  uint32_t kept = valid;
  uint64_t mass = all;
  if (P || K < valid) {
    const Leaf cut = descend(P, K);
    kept = cut.count();
    mass = cut.total();
  }
  const double u = a.draws_f64 ? static_cast<const double*>(a.draws)[m]
                               : (double)static_cast<const float*>(a.draws)[m];
  const uint64_t uf = u > 0.0 ? (u < 1.0 ? (uint64_t)(u * 18446744073709551616.0) : ~0ull) : 0;
  const Leaf d = descend(__umul64hi(uf, mass) + 1, 0xFFFFFFFFu);

  // The token of rank d.in - 1 among those of value d.key, by index: the segment of the row
  // that holds it, then its place there.
  const int seg = (V + SEGS - 1) / SEGS;
  for (int j = tid; j < SEGS; j += TT) s.kcnt[j] = 0;
  __syncthreads();
  if (listed == d.bin) {
    for (uint32_t i = tid; i < min(s.n_list, (uint32_t)LIST); i += TT)
      if (s.lkey[i] == d.key) atomicAdd(&s.kcnt[s.lidx[i] / seg], 1u);
  } else {
    for_row<DT>(row, V, [&](int i, float x) {
      if (key_of<DT>(x) == d.key) atomicAdd(&s.kcnt[i / seg], 1u);
    });
  }
  __syncthreads();
  find<NK>(s, nullptr, s.kcnt, 0, 0, 0, d.in);
  if (tid >= 64) return;
  const int i0 = (int)s.f_bin * seg, i1 = min(V, i0 + seg);
  uint32_t left = d.in - 1 - s.f_cnt;
  for (int i = i0; i < i1; i += 64) {
    const int at = i + tid;
    bool hit = false;
    if (at < i1) {
      if constexpr (DT == 2)
        hit = key_of<DT>(row[at]) == d.key;
      else
        hit = key_of<DT>(value_of<DT>(row[at])) == d.key;
    }
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

template <int DT>
int go(const TokArgs& a, hipStream_t st) {
  constexpr auto kern = sample_tokens_kernel<DT>;
  if (int rc = allow_dynamic_lds<kern, (int)sizeof(Lds)>()) return rc;
  kern<<<a.M, TT, sizeof(Lds), st>>>(a);
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
  return dtype == 0 ? go<0>(a, st) : dtype == 1 ? go<1>(a, st) : go<2>(a, st);
}

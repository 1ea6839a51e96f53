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
// M is an integer, so x k - M is one fused multiply-add with a single rounding at the
// size of its result, and sums taken against different M are brought together by exact
// powers of two. k is the float32 nearest log2(e) / T, and logp uses that same k, so its
// rounding moves logp by less than half a step of float32 and does not grow with an
// offset common to all logits. Everything per row is float64 from S on: the ratio of a
// token next to a border of the clip decides whether it has a gradient at all.
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
  float k;              // log2(e) / T
};

// What the gradient needs of a row: e_v = exp2(x_v k - M), or exp2((x_v - m) k) where M
// is not finite (rows whose logits are all below -1e30, or not finite).
struct RowStat {
  float M, S, m, pad;
};

using Policy = grpo_policy_t;

template <int DT>
__device__ __forceinline__ float load1(const void* x, int64_t i) {
  if (DT == F32) return static_cast<const float*>(x)[i];
  return e2f<DT == F16>(static_cast<const uint16_t*>(x)[i]);
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

// S, and t = sum e (x k - M) for the entropy, against an M of its own.
template <bool ENT>
struct Sums {
  float M = LOWEST, S = 0.f, t = 0.f;
  __device__ __forceinline__ void raise(float to) {  // M is an integer, to > M
    const float f = __builtin_amdgcn_exp2f(M - to);
    if (ENT) t = f * (t + (M - to) * S);
    S *= f;
    M = to;
  }
  // 32 above M is still far from the end of float32's range: M moves rarely.
  __device__ __forceinline__ void admit(float top, float k) {
    if (top * k > M + 32.f) raise(rintf(top * k));
  }
  __device__ __forceinline__ void add(float x, float k) {
    const float a = fmaf(x, k, -M), e = __builtin_amdgcn_exp2f(a);
    S += e;
    if (ENT) t = fmaf(e, fmaxf(a, -1024.f), t);  // a = -inf: 0, not 0 * inf
  }
  __device__ __forceinline__ void join(float M2, float S2, float t2) {
    if (M2 > M) raise(M2);
    const float f = __builtin_amdgcn_exp2f(M2 - M);
    if (ENT) t = fmaf(f, t2 + (M2 - M) * S2, t);
    S = fmaf(f, S2, S);
  }
};

template <int NT>
__device__ __forceinline__ float block_max(float v, float* red) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < NT / 64; ++w) v = fmaxf(v, red[w]);
  return v;
}
template <int NT>
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum_dpp(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < NT / 64; ++w) v += red[w];
  return v;
}

// The statistics of a row by one workgroup, the same in every thread.
template <int DT, bool ENT, int NT>
__device__ __forceinline__ RowStat row_stat(const void* row, int V, float k, float* red,
                                            float* ent) {
  const int head = head_of<DT>(row, V), nvec = (V - head) / PER<DT>;
  const uint4* const vec = reinterpret_cast<const uint4*>(static_cast<const char*>(row) +
                                                          (int64_t)head * SIZE<DT>);
  const int tail = head + nvec * PER<DT>;
  Sums<ENT> s;
  for (int i = threadIdx.x; i < nvec; i += NT) {
    float f[PER<DT>];
    unpack<DT>(vec[i], f);
    float top = f[0];
#pragma unroll
    for (int j = 1; j < PER<DT>; ++j) top = fmaxf(top, f[j]);
    s.admit(top, k);
#pragma unroll
    for (int j = 0; j < PER<DT>; ++j) s.add(f[j], k);
  }
  if ((int)threadIdx.x < head + V - tail) {
    const float x = load1<DT>(row, (int)threadIdx.x < head ? threadIdx.x
                                                           : tail + threadIdx.x - head);
    s.admit(x, k);
    s.add(x, k);
  }
  RowStat r;
  r.M = block_max<NT>(s.M, red);
  Sums<ENT> all;
  all.M = r.M;
  all.join(s.M, s.S, s.t);
  r.S = block_sum<NT>(all.S, red);
  const float t = ENT ? block_sum<NT>(all.t, red) : 0.f;
  r.m = 0.f;
  r.pad = 0.f;
  if (ENT) *ent = (float)(LN2 * (log2((double)r.S) - (double)t / (double)r.S));
  if (r.S > 0.f && r.S < INFINITY) return r;
  // no finite logit above -1e30, or one that is not finite: the maximum, then the sum
  float m = -INFINITY;
  for (int v = threadIdx.x; v < V; v += NT) m = fmaxf(m, load1<DT>(row, v));
  m = block_max<NT>(m, red);
  float S = 0.f, u = 0.f;
  for (int v = threadIdx.x; v < V; v += NT) {
    const float a = (load1<DT>(row, v) - m) * k, e = __builtin_amdgcn_exp2f(a);
    S += e;
    if (ENT) u = fmaf(e, fmaxf(a, -1024.f), u);
  }
  r.M = INFINITY;
  r.S = block_sum<NT>(S, red);
  r.m = m;
  if (ENT) {
    u = block_sum<NT>(u, red);
    *ent = (float)(LN2 * (log2((double)r.S) - (double)u / (double)r.S));
  }
  return r;
}

// logp of the row's token; NaN for an id outside the vocabulary.
template <int DT>
__device__ __forceinline__ double row_logp(const void* row, int64_t id, int V, float k,
                                           const RowStat& r) {
  if (id < 0 || id >= V) return __builtin_nan("");
  const double x = load1<DT>(row, id);
  const double a = r.M < INFINITY ? fma(x, (double)k, -(double)r.M) : (x - (double)r.m) * (double)k;
  return LN2 * (a - log2((double)r.S));
}

template <int DT>
__device__ __forceinline__ const void* row_at(const Rows& q, int64_t r) {
  const int64_t b = r / q.S, s = r - b * q.S;
  return static_cast<const char*>(q.x) + (b * q.sb + s * q.ss) * SIZE<DT>;
}

constexpr int NT = 512;

template <int DT, bool ENT>
__global__ void __launch_bounds__(NT) logp_kernel(Rows q, double* logp64, float* logp,
                                                  float* entropy, RowStat* stat) {
  __shared__ float red[NT / 64];
  const int64_t r = blockIdx.x;
  float ent = 0.f;
  double lp = 0.0;
  RowStat st{0.f, 1.f, 0.f, 0.f};
  if (!q.mask || q.mask[r]) {
    const void* row = row_at<DT>(q, r);
    st = row_stat<DT, ENT, NT>(row, q.V, q.k, red, &ent);
    if (threadIdx.x == 0) lp = row_logp<DT>(row, q.ids[r], q.V, q.k, st);
  }
  if (threadIdx.x == 0) {
    if (logp64) logp64[r] = lp;
    logp[r] = (float)lp;
    if (ENT) entropy[r] = ent;
    if (stat) stat[r] = st;
  }
}

// grad[r][v] = coef[r] scale / T (1[v = id] - e_v / S); scale: a device scalar or null.
template <int DT>
__global__ void __launch_bounds__(NT) logits_grad_kernel(Rows q, const RowStat* stat,
                                                         const float* coef, const float* scale,
                                                         float inv_t, void* grad) {
  const int64_t r = blockIdx.x;
  const void* row = row_at<DT>(q, r);
  char* const out = static_cast<char*>(grad) + r * q.V * SIZE<DT>;
  const int V = q.V;
  const bool on = !q.mask || q.mask[r];
  RowStat st{0.f, 1.f, 0.f, 0.f};
  float c = 0.f;
  int64_t id = -1;
  if (on) {
    st = stat[r];
    c = coef[r] * (scale ? *scale : 1.f) * inv_t;
    id = q.ids[r];
  }
  const float neg = -c / st.S, k = q.k;
  auto value = [&](float x) __attribute__((always_inline)) {
    const float a = st.M < INFINITY ? fmaf(x, k, -st.M) : (x - st.m) * k;
    return __builtin_amdgcn_exp2f(a) * neg;
  };
  const int head = head_of<DT>(out, V), nvec = (V - head) / PER<DT>, tail = head + nvec * PER<DT>;
  const char* const src = static_cast<const char*>(row) + (int64_t)head * SIZE<DT>;
  uint4* const dst = reinterpret_cast<uint4*>(out + (int64_t)head * SIZE<DT>);
  const bool same = aligned16(src);
  for (int i = threadIdx.x; i < nvec; i += NT) {
    float f[PER<DT>];
    if (on) {
      if (same) {
        unpack<DT>(reinterpret_cast<const uint4*>(src)[i], f);
      } else {
#pragma unroll
        for (int j = 0; j < PER<DT>; ++j) f[j] = load1<DT>(src, (int64_t)i * PER<DT> + j);
      }
#pragma unroll
      for (int j = 0; j < PER<DT>; ++j) {
        const int64_t v = head + (int64_t)i * PER<DT> + j;
        f[j] = value(f[j]) + (v == id ? c : 0.f);
      }
    } else {
#pragma unroll
      for (int j = 0; j < PER<DT>; ++j) f[j] = 0.f;
    }
    dst[i] = pack<DT>(f);
  }
  if ((int)threadIdx.x < head + V - tail) {
    const int v = (int)threadIdx.x < head ? threadIdx.x : tail + threadIdx.x - head;
    store1<DT>(out, v, on ? value(load1<DT>(row, v)) + (v == id ? c : 0.f) : 0.f);
  }
}

// ------------------------------------------------------------- policy loss --

// Counted tokens of each sequence.
__global__ void __launch_bounds__(256) count_kernel(const uint8_t* mask, int S, int* counts) {
  __shared__ float red[4];
  const uint8_t* m = mask + (int64_t)blockIdx.x * S;
  int n = 0;
  for (int s = threadIdx.x; s < S; s += 256) n += m[s] != 0;
  // at most 2^31 tokens of a sequence, summed as two exact float32 halves
  const float lo = block_sum<256>((float)(n & 4095), red);
  const float hi = block_sum<256>((float)(n >> 12), red);
  if (threadIdx.x == 0) counts[blockIdx.x] = (int)hi * 4096 + (int)lo;
}

struct Tokens {
  const double* logp64;  // [R], or null: logp
  const float* logp;     // [R]
  const float* old;      // [R] or null: logp itself
  const float* ref;      // [R] or null
  const float* adv;      // [B], or [R] (adv_tokens)
  const uint8_t* mask;   // [R] or null
  const int* counts;     // [B] or null: S each
  int B, S;
  bool adv_tokens;
};

// Sums over the counted tokens: w l, then r, stopped tokens, KL and old - logp.
struct TokenSums {
  double v[5];
};

// Counted tokens and sequences of the batch, the same in every thread.
template <int NT_>
__device__ __forceinline__ void totals(const Tokens& t, double* red, double* tokens,
                                       double* seqs) {
  double n = 0.0, q = 0.0;
  if (!t.counts) {
    *tokens = (double)t.B * t.S;
    *seqs = t.B;
    return;
  }
  for (int b = threadIdx.x; b < t.B; b += NT_) {
    const int c = t.counts[b];
    n += c;
    q += c > 0;
  }
  for (int o = 32; o; o >>= 1) {
    n += __shfl_xor(n, o);
    q += __shfl_xor(q, o);
  }
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
  __syncthreads();
  *tokens = n;
  *seqs = q;
}

__device__ __forceinline__ double token_weight(const Policy& p, int in_row, double tokens,
                                               double seqs) {
  if (p.normalizer == 0) return 1.0 / tokens;
  if (p.normalizer == 1) return 1.0 / (in_row * seqs);
  return 1.0 / p.denom;
}

// One counted token: d loss / d logp, its terms added to s.
__device__ __forceinline__ double token_loss(const Policy& p, double lp, double old, bool has_ref,
                                             double ref, double a, double w, TokenSums& s) {
  const double r = exp(lp - old);
  const double lo = 1.0 - p.eps_low, hi = 1.0 + p.eps_high, cap = p.delta;
  const double clipped = fmin(fmax(r, lo), hi);
  const double free_gain = fmin(r, cap) * a, clip_gain = clipped * a;
  // whether the smaller gain moves with r
  const bool follows = (free_gain <= clip_gain && r <= cap) ||
                       (clip_gain <= free_gain && clipped == r);
  double l = -fmin(free_gain, clip_gain), d = follows ? -r * a : 0.0, kl = 0.0;
  if (r != r || a != a) l = d = r * a;  // fmin would hide a NaN
  if (has_ref) {
    const double q = ref - lp, e = exp(q);
    kl = e - q - 1.0;
    l += p.beta * kl;
    d += p.beta * (1.0 - e);
  }
  s.v[0] += w * l;
  s.v[1] += r;
  s.v[2] += follows ? 0.0 : 1.0;
  s.v[3] += kl;
  s.v[4] += old - lp;
  return d * w;
}

__device__ __forceinline__ double token_at(const Policy& p, const Tokens& t, int64_t r,
                                           double tokens, double seqs, TokenSums& s) {
  if (t.mask && !t.mask[r]) return 0.0;
  const int b = (int)(r / t.S);
  const double lp = t.logp64 ? t.logp64[r] : (double)t.logp[r];
  const double w = token_weight(p, t.counts ? t.counts[b] : t.S, tokens, seqs);
  return token_loss(p, lp, t.old ? (double)t.old[r] : lp, t.ref != nullptr,
                    t.ref ? (double)t.ref[r] : 0.0, t.adv[t.adv_tokens ? r : b], w, s);
}

// The workgroup's sums, in wave order (thread 0 writes them).
template <int NT_>
__device__ __forceinline__ void write_sums(TokenSums s, double* red, double* out) {
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    double v = s.v[i];
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
      v = red[0];
      for (int w = 1; w < NT_ / 64; ++w) v += red[w];
      out[i] = v;
    }
  }
}

// coef (null: none): d loss / d logp of every token, 0 where not counted.
__global__ void __launch_bounds__(256) policy_kernel(Policy p, Tokens t, float* coef,
                                                     const float* scale, double* sums) {
  __shared__ double red[8];
  double tokens, seqs;
  totals<256>(t, red, &tokens, &seqs);
  const int64_t R = (int64_t)t.B * t.S;
  const double g = scale ? *scale : 1.0;
  TokenSums s{};
  for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < R; r += (int64_t)gridDim.x * 256) {
    const double d = token_at(p, t, r, tokens, seqs, s);
    if (coef) coef[r] = (float)(d * g);
  }
  if (sums) write_sums<256>(s, red, sums + 5 * (int64_t)blockIdx.x);
}

// loss and metrics from the workgroups' sums, in their order.
__global__ void __launch_bounds__(256) finish_kernel(Tokens t, const double* sums, int blocks,
                                                     float* loss, float* metrics) {
  __shared__ double red[8], out[5];
  double tokens, seqs;
  totals<256>(t, red, &tokens, &seqs);
  TokenSums s{};
  for (int i = threadIdx.x; i < blocks; i += 256)
    for (int j = 0; j < 5; ++j) s.v[j] += sums[5 * i + j];
  write_sums<256>(s, red, out);
  if (threadIdx.x) return;
  *loss = (float)out[0];
  for (int j = 0; j < 4; ++j) metrics[j] = tokens > 0.0 ? (float)(out[1 + j] / tokens) : 0.f;
}

// ----------------------------------------------------------------- host --

// Workspace of the loss entry points: counted tokens per sequence, the workgroups'
// sums, and (from logits) the float64 log-probabilities.
constexpr int SUM_BLOCKS = 256;
struct PolicyWs {
  size_t counts, sums, logp64, total;
};
PolicyWs policy_ws(int B, int S, bool logits) {
  PolicyWs w{};
  size_t o = 0;
  auto take = [&](size_t n) {
    const size_t at = o;
    o += (n + 255) / 256 * 256;
    return at;
  };
  w.counts = take((size_t)B * 4);
  w.sums = take(SUM_BLOCKS * 5 * 8);
  w.logp64 = take(logits ? (size_t)B * S * 8 : 0);
  w.total = o;
  return w;
}

int batch_check(int B, int S) {
  if (B < 0 || S < 0) return einval("negative dimension");
  if ((int64_t)B * S >= (1ll << 31) || B >= (1 << 23)) return einval("too many tokens");
  return GRPO_OK;
}

int rows_check(const void* x, int dtype, int64_t sb, int64_t ss, int B, int S, int V,
               const int64_t* ids, float temperature) {
  if (int rc = batch_check(B, S)) return rc;
  if ((int64_t)B * S >= (1 << 22)) return einval("2^22 rows of logits or more");
  if (V < 1) return einval("an empty vocabulary");
  if (dtype < 0 || dtype > 2) return einval("dtype must be 0 (bf16), 1 (float16) or 2 (float32)");
  if (!(temperature > 0.f) || !(temperature < INFINITY))
    return einval("temperature must be positive and finite");
  const float k = (float)(1.0 / LN2 / (double)temperature);
  if (!(k >= 1e-30f) || !(k <= 1e30f)) return einval("temperature out of range");
  if ((int64_t)B * S == 0) return GRPO_OK;
  if (!x || !ids) return einval("null pointer");
  if (sb < 0 || ss < 0) return einval("negative row stride");
  const int size = dtype == F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(x) % size) return einval("logits are not aligned to their type");
  return GRPO_OK;
}

Rows rows_of(const void* x, int64_t sb, int64_t ss, int S, int V, const int64_t* ids,
             const uint8_t* mask, float temperature) {
  return Rows{x, sb, ss, S, V, ids, mask, (float)(1.0 / LN2 / (double)temperature)};
}

template <int DT>
int launch_logp(const Rows& q, int64_t R, double* logp64, float* logp, float* entropy,
                RowStat* stat, hipStream_t st) {
  if (entropy) logp_kernel<DT, true><<<(unsigned)R, NT, 0, st>>>(q, logp64, logp, entropy, stat);
  else logp_kernel<DT, false><<<(unsigned)R, NT, 0, st>>>(q, logp64, logp, entropy, stat);
  return launch_check("token_logprobs");
}

int run_logp(int dtype, const Rows& q, int64_t R, double* logp64, float* logp, float* entropy,
             RowStat* stat, hipStream_t st) {
  if (dtype == BF16) return launch_logp<BF16>(q, R, logp64, logp, entropy, stat, st);
  if (dtype == F16) return launch_logp<F16>(q, R, logp64, logp, entropy, stat, st);
  return launch_logp<F32>(q, R, logp64, logp, entropy, stat, st);
}

int run_grad(int dtype, const Rows& q, int64_t R, const RowStat* stat, const float* coef,
             const float* scale, float temperature, void* grad, hipStream_t st) {
  const float inv_t = 1.f / temperature;
  const unsigned n = (unsigned)R;
  if (dtype == BF16)
    logits_grad_kernel<BF16><<<n, NT, 0, st>>>(q, stat, coef, scale, inv_t, grad);
  else if (dtype == F16)
    logits_grad_kernel<F16><<<n, NT, 0, st>>>(q, stat, coef, scale, inv_t, grad);
  else
    logits_grad_kernel<F32><<<n, NT, 0, st>>>(q, stat, coef, scale, inv_t, grad);
  return launch_check("token_logprobs_backward");
}

int policy_check(const grpo_policy_t* p, int B, int S, const float* adv, const void* ws,
                 size_t ws_bytes, bool logits) {
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
  if (ws_bytes < policy_ws(B, S, logits).total) {
    set_error("workspace too small");
    return GRPO_EWORKSPACE;
  }
  return GRPO_OK;
}

// Counts, then the tokens' losses and derivatives, then the sums' end.
int run_policy(const Policy& p, Tokens t, char* ws, const PolicyWs& o, float* coef, float* loss,
               float* metrics, hipStream_t st) {
  const int64_t R = (int64_t)t.B * t.S;
  if (t.mask && R) {
    int* counts = reinterpret_cast<int*>(ws + o.counts);
    count_kernel<<<(unsigned)t.B, 256, 0, st>>>(t.mask, t.S, counts);
    if (int rc = launch_check("policy_count")) return rc;
    t.counts = counts;
  }
  double* sums = reinterpret_cast<double*>(ws + o.sums);
  const int blocks = (int)(R ? cdiv(R, 256) < SUM_BLOCKS ? cdiv(R, 256) : SUM_BLOCKS : 0);
  if (blocks) {
    policy_kernel<<<blocks, 256, 0, st>>>(p, t, coef, nullptr, sums);
    if (int rc = launch_check("policy_loss")) return rc;
  }
  finish_kernel<<<1, 256, 0, st>>>(t, sums, blocks, loss, metrics);
  return launch_check("policy_finish");
}

}  // namespace

extern "C" int grpo_token_logprobs(const void* logits, int dtype, int64_t stride_b,
                                   int64_t stride_s, int B, int S, int V, const int64_t* ids,
                                   const uint8_t* mask, float temperature, float* logp,
                                   float* entropy, float* stat, grpo_stream_t stream) {
  if (int rc = rows_check(logits, dtype, stride_b, stride_s, B, S, V, ids, temperature)) return rc;
  const int64_t R = (int64_t)B * S;
  if (!R) return GRPO_OK;
  if (!logp) return einval("null pointer");
  if (!aligned16(stat)) return einval("stat must be 16-byte aligned");
  return run_logp(dtype, rows_of(logits, stride_b, stride_s, S, V, ids, mask, temperature), R,
                  nullptr, logp, entropy, reinterpret_cast<RowStat*>(stat), as_stream(stream));
}

extern "C" int grpo_token_logprobs_backward(const void* logits, int dtype, int64_t stride_b,
                                            int64_t stride_s, int B, int S, int V,
                                            const int64_t* ids, const uint8_t* mask,
                                            float temperature, const float* stat,
                                            const float* grad_logp, const float* scale,
                                            void* grad_logits, grpo_stream_t stream) {
  if (int rc = rows_check(logits, dtype, stride_b, stride_s, B, S, V, ids, temperature)) return rc;
  const int64_t R = (int64_t)B * S;
  if (!R) return GRPO_OK;
  if (!stat || !grad_logp || !grad_logits) return einval("null pointer");
  if (!aligned16(stat)) return einval("stat must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(grad_logits) % (dtype == F32 ? 4 : 2))
    return einval("grad_logits is not aligned to its type");
  return run_grad(dtype, rows_of(logits, stride_b, stride_s, S, V, ids, mask, temperature), R,
                  reinterpret_cast<const RowStat*>(stat), grad_logp, scale, temperature,
                  grad_logits, as_stream(stream));
}

extern "C" size_t grpo_policy_loss_workspace_bytes(int B, int S, int from_logits) {
  return B < 0 || S < 0 ? 0 : policy_ws(B, S, from_logits != 0).total;
}

extern "C" int grpo_policy_loss(const float* logp, const float* old_logp, const float* ref_logp,
                                const float* advantages, int adv_tokens, const uint8_t* mask,
                                int B, int S, const grpo_policy_t* policy, float* loss,
                                float* metrics, void* workspace, size_t workspace_bytes,
                                grpo_stream_t stream) {
  if (int rc = policy_check(policy, B, S, advantages, workspace, workspace_bytes, false)) return rc;
  if (((int64_t)B * S && !logp) || !loss || !metrics) return einval("null pointer");
  Tokens t{nullptr, logp, old_logp, ref_logp, advantages, mask, nullptr, B, S, adv_tokens != 0};
  return run_policy(*policy, t, static_cast<char*>(workspace), policy_ws(B, S, false),
                    nullptr, loss, metrics, as_stream(stream));
}

extern "C" int grpo_policy_loss_backward(const float* logp, const float* old_logp,
                                         const float* ref_logp, const float* advantages,
                                         int adv_tokens, const uint8_t* mask, int B, int S,
                                         const grpo_policy_t* policy, const float* grad_loss,
                                         float* grad_logp, void* workspace,
                                         size_t workspace_bytes, grpo_stream_t stream) {
  if (int rc = policy_check(policy, B, S, advantages, workspace, workspace_bytes, false)) return rc;
  const int64_t R = (int64_t)B * S;
  if (!R) return GRPO_OK;
  if (!logp || !grad_loss || !grad_logp) return einval("null pointer");
  hipStream_t st = as_stream(stream);
  Tokens t{nullptr, logp, old_logp, ref_logp, advantages, mask, nullptr, B, S, adv_tokens != 0};
  if (mask) {  // the forward's counts, in the same workspace
    t.counts = reinterpret_cast<const int*>(static_cast<char*>(workspace) +
                                            policy_ws(B, S, false).counts);
  }
  const int blocks = (int)(cdiv(R, 256) < 2048 ? cdiv(R, 256) : 2048);
  policy_kernel<<<blocks, 256, 0, st>>>(*policy, t, grad_logp, grad_loss, nullptr);
  return launch_check("policy_loss_backward");
}

extern "C" int grpo_policy_loss_logits(const void* logits, int dtype, int64_t stride_b,
                                       int64_t stride_s, int B, int S, int V, const int64_t* ids,
                                       const uint8_t* mask, float temperature,
                                       const float* old_logp, const float* ref_logp,
                                       const float* advantages, int adv_tokens,
                                       const grpo_policy_t* policy, float* loss, float* logp,
                                       float* metrics, float* stat, float* coef, void* workspace,
                                       size_t workspace_bytes, grpo_stream_t stream) {
  if (int rc = rows_check(logits, dtype, stride_b, stride_s, B, S, V, ids, temperature)) return rc;
  if (int rc = policy_check(policy, B, S, advantages, workspace, workspace_bytes, true)) return rc;
  const int64_t R = (int64_t)B * S;
  if ((R && !logp) || !loss || !metrics) return einval("null pointer");
  if ((stat == nullptr) != (coef == nullptr)) return einval("stat and coef go together");
  if (!aligned16(stat)) return einval("stat must be 16-byte aligned");
  hipStream_t st = as_stream(stream);
  char* const ws = static_cast<char*>(workspace);
  const PolicyWs o = policy_ws(B, S, true);
  double* const lp = reinterpret_cast<double*>(ws + o.logp64);
  if (R) {
    const Rows q = rows_of(logits, stride_b, stride_s, S, V, ids, mask, temperature);
    if (int rc = run_logp(dtype, q, R, lp, logp, nullptr, reinterpret_cast<RowStat*>(stat), st))
      return rc;
  }
  Tokens t{lp, logp, old_logp, ref_logp, advantages, mask, nullptr, B, S, adv_tokens != 0};
  return run_policy(*policy, t, ws, o, coef, loss, metrics, st);
}

// Paged GQA attention of a tree of drafted tokens (grpo_paged_tree_attn), gfx950: T nodes per
// sequence whose keys and values stand in the cache's slots after its context_lens[b] tokens;
// node i attends those tokens, its ancestors and itself. What the reference's decode attention
// (src/triton_kernels/paged_kv.py:63-251) does for one token, for a tree of them.
//
// A token that a node does not attend is not read for it: whatever stands there (NaN of a slot
// never written, another branch) stays out. A node that attends nothing gets 0.
#include <algorithm>
#include <cmath>

#include "lds_dma.hpp"
#include "tree.hpp"

using namespace grpo;

namespace {

constexpr int GT = 256;  // threads of the plain kernel
constexpr int GD = 512;  // its largest head dim
constexpr float LOG2E = 1.4426950408889634f;

struct TreeArgs {
  const uint16_t* q;
  int64_t qsb, qst, qsh;
  const uint16_t* kc;
  const uint16_t* vc;
  Pages pages;
  const int32_t* cl;
  const int32_t* parents;  // or null: a chain
  int64_t ps;
  const int32_t* counts;
  uint16_t* out;  // [B][T][Hq][D]
  int B, T, Hq, D;
  float scale;
};

// What node lane sees of the tree, in every wave (lane < T).
__device__ __forceinline__ uint64_t sees(const TreeArgs& a, int b) {
  const int lane = threadIdx.x & 63;
  if (!a.parents) return lane == 63 ? ~0ull : (2ull << lane) - 1;
  const int p = lane < a.T ? node_parent(a.parents[(int64_t)b * a.ps + lane], lane) : -1;
  return ancestors(p);
}

// A workgroup per (node, query head): 256 tokens at a time, a score per thread, then the
// threads over the dims. For the head dims and addresses that the MFMA kernel does not take.
template <bool F16>
__global__ void __launch_bounds__(GT) tree_attn_plain_kernel(TreeArgs a) {
  __shared__ float qs[GD], pr[GT], red[GT / 64];
  __shared__ int64_t rows[GT];
  const int b = blockIdx.x / a.T, t = blockIdx.x - b * a.T, h = blockIdx.y, tid = threadIdx.x;
  const int D = a.D, Hkv = a.pages.Hkv, kvh = h / (a.Hq / Hkv);
  uint16_t* const out = a.out + ((int64_t)blockIdx.x * a.Hq + h) * D;
  const int context = a.cl[b];
  const bool used = t < nodes_of(a.counts, b, a.T, context);
  const uint64_t all = sees(a, b);
  const uint64_t mask = (uint64_t)__shfl((long long)all, t);
  const int64_t head = (int64_t)kvh * a.pages.block_size;
  const uint16_t* const q = a.q + (int64_t)b * a.qsb + (int64_t)t * a.qst + (int64_t)h * a.qsh;
  for (int d = tid; d < D; d += GT) qs[d] = e2f<F16>(q[d]);
  // (no further than the table: a length past it would be walked for seconds)
  const int64_t cap = (int64_t)a.pages.max_blocks * a.pages.block_size;
  const int64_t last = used ? min((int64_t)context + t + 1, cap) : 0;
  float m_run = -INFINITY, l_run = 0.f, acc[GD / GT] = {};
  for (int64_t t0 = 0; t0 < last; t0 += GT) {
    __syncthreads();
    const int64_t slot = t0 + tid;
    const int64_t node = slot - context;
    const bool on = slot < last && (node < 0 || ((mask >> node) & 1));
    const int64_t row = on ? a.pages.row(b, slot) : -1;
    float s = -INFINITY;
    if (row >= 0) {
      const uint16_t* const k = a.kc + (row + head) * D;
      s = 0.f;
      for (int d = 0; d < D; ++d) s = fmaf(qs[d], e2f<F16>(k[d]), s);
      s *= a.scale * LOG2E;
    }
    float top = s;
    for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    if ((tid & 63) == 0) red[tid >> 6] = top;
    __syncthreads();
    for (int w = 0; w < GT / 64; ++w) top = fmaxf(top, red[w]);
    const float m_new = fmaxf(m_run, top), m_use = m_new == -INFINITY ? 0.f : m_new;
    const float corr = exp2f(m_run - m_use);
    rows[tid] = row;
    pr[tid] = exp2f(s - m_use);
    __syncthreads();
    m_run = m_new;
    l_run *= corr;
#pragma unroll
    for (int i = 0; i < GD / GT; ++i) acc[i] *= corr;
    for (int j = 0; j < GT; ++j) {
      if (rows[j] < 0) continue;
      const float p = pr[j];
      l_run += p;
      const uint16_t* const v = a.vc + (rows[j] + head) * D;
#pragma unroll
      for (int i = 0; i < GD / GT; ++i)
        if (tid + i * GT < D) acc[i] = fmaf(p, e2f<F16>(v[tid + i * GT]), acc[i]);
    }
  }
  const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
#pragma unroll
  for (int i = 0; i < GD / GT; ++i)
    if (tid + i * GT < D) out[tid + i * GT] = f2e<F16>(l_run == 0.f ? 0.f : acc[i] * inv);
}

// ------------------------------------------------------------ MFMA kernel --
// The T (Hq / Hkv) rows (node, head of the group) of one KV head are the columns of 32x32x16
// MFMAs, so that K and V are read once for all of them:
//  * A wave owns 32 rows. A workgroup has RW waves side by side on rows times 8 / RW on tokens,
//    which take the 32-token parts of each step and meet in LDS at the end. A sequence's tokens
//    are cut over workgroups, one per CU, where there are few of them (a second kernel joins the
//    parts).
//  * K and V of a step come to LDS by loads of their own, RING - 1 steps ahead (96 KiB on their
//    way per CU). The cache rows of WIN tokens stand in LDS too.
//  * S^T = K Q^T leaves lane (row ln, half lh) with 16 of 32 tokens' scores of its row, which
//    are the operand P^T of O^T = V^T P^T if its contraction index (lh, e) of product j means
//    token 16 j + 8 (e / 4) + 4 lh + e % 4: P never leaves the lane. V is turned as it is read
//    from LDS.
//  * The scores of the next tile are made between the weights of this one: on a SIMD a product
//    takes 32 cycles, an exponential 16, another instruction 4, side by side.
//  * P is two 16-bit values, a weight's rounding and the rest's (2^-17 of the weight off in bf16,
//    2^-22 in float16), as in the decode attention: V times each is summed in float32. One value
//    alone would add as much error as the rounding of the result, 0.0022 against 0.0017 of it in
//    bf16, for 117 instead of 150 us (64 trees of 32, 2500 tokens), 50 instead of 62 (one of 61, 30
//    thousand), 26 instead of 28.6 (32 of 16, 1500). In float16 a row's largest weight is 2^12 or
//    more, so that what a small one loses below 2^-24 is 2^-37 of the largest: a long tail of faint
//    tokens beside one that stands out keeps its mass.
//  * Steps that reach past the cached tokens, or a window that holds a missing block, have V
//    cleaned in LDS first and the scores masked: the same loop adds them, so that O stays in one
//    set of registers.
// Measured at 28 and 4 heads of 128 dims, blocks of 16, contexts of half to one and a half times
// the mean: 64 trees of 4 nodes over 2500 tokens 88 us (3.8 TB/s: the reading of the cache), 64
// of 32 150 us (361 MB, 74 GFLOP), one of 61 over 30 thousand 62 us, 64 of 32 and 64 dims 102 us.
// With many rows the two waves of a SIMD take 2.5 thousand cycles for a tile each, of which 1536 are
// products, and the longest sequence ends last. (With P in one value: equal shares of all tokens for
// every workgroup instead, of up to three sequences each, 164 against 146 us, the parts' sums are 60
// MB; second parts of the longest sequences only, 143 against 119; 105 of 119 us without any
// reading of the cache.)

constexpr int WIN = 4096;        // tokens whose cache rows stand in LDS at a time
constexpr int RING = 4;          // steps of K and V that stand there
constexpr int MAX_SPLITS = 64;
constexpr int LEAST_CHUNK = 128; // tokens of a split at least

typedef float f32x16_t __attribute__((ext_vector_type(16)));

struct FastArgs {
  TreeArgs t;
  int splits, RP;  // RP: rows of a (sequence, KV head) in the workspace
  float* ws_o;     // [B][Hkv][splits][RP][D]
  float* ws_ml;    // [B][Hkv][splits][RP][2]: max (log2 domain), sum
};

template <bool F16>
__device__ __forceinline__ f32x16_t mfma32(uint4 a, uint4 b, f32x16_t c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
}

// 16 bytes per lane from a 64-bit address of its own to 1 KiB at the wave-uniform LDS address
// lds (see lds_dma.hpp).
__device__ __forceinline__ void dma16_at(uint32_t lds, const void* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p)
               : "memory");
}

// The tokens of sequence b and how they are cut: split z takes [z chunk, (z + 1) chunk).
struct Cut {
  int context, nodes, total, chunk, splits;
};
__device__ __forceinline__ Cut cut_of(const TreeArgs& a, int len, int count, int splits, int step) {
  Cut c;
  const int cap = a.pages.max_blocks * a.pages.block_size;
  c.nodes = len < 0 ? 0 : min(max(count, 0), a.T);
  c.context = min(max(len, 0), cap);
  c.total = c.nodes ? c.context + min(c.nodes, cap - c.context) : 0;
  const uint32_t part = ((uint32_t)c.total + splits - 1) / (uint32_t)splits;
  c.chunk = max((int)((part + step - 1) / step) * step, LEAST_CHUNK);
  c.splits = ((uint32_t)c.total + c.chunk - 1) / (uint32_t)c.chunk;
  return c;
}

// All ones in the halves of d that are an infinity or NaN (exponent bits all set).
template <bool F16>
__device__ __forceinline__ uint32_t inf_halves(uint32_t d) {
  constexpr uint32_t X = F16 ? 0x7C00u : 0x7F80u;
  return ((d & X) == X ? 0xFFFFu : 0u) | ((d & (X << 16)) == X << 16 ? 0xFFFF0000u : 0u);
}

// Four 16-bit values per lane, turned: of 16 lanes' rows 0 to 3, which lanes 4 r to 4 r + 3 name
// with an address for four values each, lane n gets value n of each.
__device__ __forceinline__ uint2 turned(const char* p) {
  typedef short s16x4_t __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) s16x4_t*)p));
}

// LDS: pieces of 1 KiB, each an instruction's, 16 bytes apart so that four (eight) of them start
// in different banks. Within one a token's 16-byte chunk c stands at c ^ swizzle(token).
template <int D>
constexpr int TPP = 512 / D;  // tokens of a piece
constexpr int PIECE = 1024 + 16;
template <int D>
constexpr int TILE = 32 / TPP<D> * PIECE;  // 32 tokens
template <int D>
__device__ __forceinline__ int swizzle(int token) {
  return D == 128 ? (token & 3) * 4 : token & 6;
}

// Of a step's tokens a wave has one tile of 32 or two.
template <int RW>
constexpr int TILES = RW == 8 ? 2 : 1;
template <int RW>
constexpr int step_of() { return 32 * TILES<RW> * (8 / RW); }

template <bool F16, int D, int RW>
__global__ void __launch_bounds__(512) tree_attn_kernel(FastArgs f) {
  constexpr int W = 8, TW = W / RW, PT = TILES<RW>, PTOK = 32 * PT, STEP = step_of<RW>();
  constexpr int ROWB = 2 * D, NCH = D / 8;            // bytes and 16-byte chunks of a row
  constexpr int TILE_B = TILE<D>, HALF_B = PT * TILE_B;
  constexpr int PART_B = 2 * HALF_B, STEP_B = TW * PART_B;
  constexpr int PPK = PTOK / TPP<D>;                  // pieces of K
  constexpr int PIECES = 2 * PPK * TW, LD = PIECES / W;
  static_assert(PIECES % W == 0, "every wave loads as many pieces");
  constexpr int KS = D / 16, DT = D / 32;             // steps of K, tiles of V
  constexpr int XCH = 2 + 16 * DT;                      // values per lane in the waves' merge
  static_assert((TW - 1) * RW * XCH * 256 <= RING * STEP_B, "the merge fits the ring");
  extern __shared__ __align__(16) char lds[];           // [RING][STEP_B], then WIN rows
  int* const rows = reinterpret_cast<int*>(lds + RING * STEP_B);
  const TreeArgs& a = f.t;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part = wave / RW, ln = lane & 31, lh = lane >> 5;
  const int Hkv = a.pages.Hkv, G = a.Hq / Hkv, R = a.T * G;
  const int pair = blockIdx.x / f.splits, split = blockIdx.x - pair * f.splits;
  const int b = pair / Hkv, kvh = pair - b * Hkv;
  if (b >= a.B) return;
  // What does not depend on the sequence's length is asked for together with it.
  const int len = a.cl[b], count = a.counts ? a.counts[b] : a.T;
  const int row0 = (blockIdx.y * RW + wave % RW) * 32, row = row0 + ln, rowc = min(row, R - 1);
  const int node = rowc / G, head = kvh * G + rowc - node * G;
  int up = lane - 1;
  if (a.parents) up = lane < a.T ? a.parents[(int64_t)b * a.ps + lane] : -1;
  uint4 qf[KS];
  {
    const uint16_t* const q =
        a.q + (int64_t)b * a.qsb + (int64_t)node * a.qst + (int64_t)head * a.qsh + 8 * lh;
#pragma unroll
    for (int i = 0; i < KS; ++i) qf[i] = *reinterpret_cast<const uint4*>(q + 16 * i);
  }
  const Cut c = cut_of(a, len, count, f.splits, STEP);
  if (split >= max(c.splits, 1)) return;
  const float sl2 = fmaxf(fabsf(a.scale) * LOG2E, 1e-30f);  // (-inf stays -inf)
  const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
  uint64_t mask = 0;  // the nodes that row ln's node attends
  const int begin = split * c.chunk, end = min(c.total, begin + c.chunk);

  const uint32_t lbase = lds_address(lds);
  // Where a block of the cache holds whole pieces, a piece is 1 KiB of it.
  const bool by_piece = a.pages.block_size % TPP<D> == 0;
  const uint32_t piece_at =
      lane / NCH * ROWB + 16 * ((lane & (NCH - 1)) ^ swizzle<D>(lane / NCH));
  auto fetch = [&](int s) __attribute__((always_inline)) {
    if (by_piece) {  // piece i's first row in lane i
      const int pc = wave + W * (lane % LD);
      const int first = rows[s * STEP + PTOK * (pc / (2 * PPK)) + (pc & (PPK - 1)) * TPP<D>];
#pragma unroll
      for (int i = 0; i < LD; ++i) {
        const int pi = wave + W * i, r = max(__builtin_amdgcn_readlane(first, i), 0);
        const uint16_t* const base = (pi / PPK) & 1 ? a.vc : a.kc;
        dma16(lbase + (s % RING) * STEP_B + pi * PIECE, piece_at, base + (int64_t)r * D);
      }
      return;
    }
    int l = lane;
    asm volatile("" : "+v"(l));
    int r[LD];
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const int pc = wave + W * i, tok = (pc & (PPK - 1)) * TPP<D> + l / NCH;
      r[i] = rows[s * STEP + PTOK * (pc / (2 * PPK)) + tok];
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const int pc = wave + W * i, tok = (pc & (PPK - 1)) * TPP<D> + l / NCH;
      const uint16_t* const base = (pc / PPK) & 1 ? a.vc : a.kc;
      dma16_at(lbase + (s % RING) * STEP_B + pc * PIECE,  // (a missing one reads row 0)
               base + (int64_t)max(r[i], 0) * D + 8 * ((l & (NCH - 1)) ^ swizzle<D>(tok)));
    }
  };

  float m_run = -INFINITY, l_run = 0.f;  // of row ln
  f32x16_t oacc[DT];  // O[ln][32 t + 8 (i / 4) + 4 lh + i % 4] in oacc[t][i]
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) oacc[t][i] = 0.f;
  // Where a lane's operands stand in a tile, less what is the same for all lanes: of K product
  // KS / 4 i's, of V those of dims from 32 t on.
  int ka[4], va[DT];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    ka[i] = ln / TPP<D> * PIECE + ln % TPP<D> * ROWB +
            16 * ((NCH / 4 * i ^ swizzle<D>(ln)) + lh);
#pragma unroll
  for (int t = 0; t < DT; ++t) {
    const int tok = 4 * lh + lane % 16 / 4, chunk = 4 * t + ln / 16 * 2 + lane % 4 / 2;
    va[t] = tok / TPP<D> * PIECE + tok % TPP<D> * ROWB + 16 * (chunk ^ swizzle<D>(tok)) +
            lane % 2 * 8;
  }
  auto k_of = [&](const char* kt, int i) __attribute__((always_inline)) {
    return *reinterpret_cast<const uint4*>(kt + ka[i / (KS / 4)] + 32 * (i % (KS / 4)));
  };
  // S^T of 32 tokens, tile q of step s.
  auto scores = [&](int s, int q) __attribute__((always_inline)) {
    const char* const kt = lds + (s % RING) * STEP_B + part * PART_B + q * TILE_B;
    f32x16_t sc;
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = 0.f;
#pragma unroll
    for (int i = 0; i < KS; ++i) sc = mfma32<F16>(k_of(kt, i), qf[i], sc);
    return sc;
  };
  // V^T of half of them (product j): of dim 32 t + ln token 16 j + 8 (e / 4) + 4 lh + e % 4 as
  // value e of v[t].
  auto values = [&](const char* vt, int j, uint4 (&v)[DT]) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      const uint2 x = turned(vt + va[t] + 16 * j / TPP<D> * PIECE);
      const uint2 y = turned(vt + va[t] + (16 * j + 8) / TPP<D> * PIECE);
      v[t] = make_uint4(x.x, x.y, y.x, y.y);
    }
  };
  // V of a step that some row does not attend as a whole: a missing token's row is 0, and so is a
  // value that is not finite in a token that not every row attends, which would be NaN times 0
  // (it is looked at again in the end).
  bool odd = false;
  auto clean = [&](int s, int t0) __attribute__((always_inline)) {
    constexpr int N = STEP * NCH / (64 * W);
    bool any = false;
    int r[N];
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = rows[s * STEP + (tid + 64 * W * i) / NCH];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int tok = (tid + 64 * W * i) / NCH, at = tok % PTOK;
      uint4* const d = reinterpret_cast<uint4*>(lds + (s % RING) * STEP_B + tok / PTOK * PART_B +
                                                HALF_B + at / TPP<D> * PIECE + at % TPP<D> * ROWB) +
                       tid % NCH;
      if (r[i] < 0) {
        *d = make_uint4(0u, 0u, 0u, 0u);
      } else if (t0 + tok >= c.context) {
        uint4 v = *d;
        const uint4 x = make_uint4(inf_halves<F16>(v.x), inf_halves<F16>(v.y),
                                   inf_halves<F16>(v.z), inf_halves<F16>(v.w));
        if (x.x | x.y | x.z | x.w) {
          v.x &= ~x.x, v.y &= ~x.y, v.z &= ~x.z, v.w &= ~x.w;
          *d = v;
          any = true;
        }
      }
    }
    odd |= __syncthreads_or(any) != 0;
  };
  // The running maximum less FIRST (room below for float16's small weights), ahead of scores up to
  // top. It stands still while they are less than MOST above it: the weights stay below 2^MOST, and
  // the sums need no factor.
  constexpr float FIRST = F16 ? 12.f : 0.f, MOST = F16 ? 15.f : 8.f;
  auto rescale = [&](float top) __attribute__((always_inline)) {
    const bool up = top > m_run + MOST;  // (the first score that is not -inf too)
    if (__ballot(up)) {
      const float m_new = up ? top - FIRST : m_run;
      const float corr = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
      l_run *= corr;
#pragma unroll
      for (int t = 0; t < DT; ++t) oacc[t] *= corr;
      m_run = m_new;
    }
  };
  auto weight = [&](float x) __attribute__((always_inline)) {
    const float m_use = m_run == -INFINITY ? 0.f : m_run;  // no token yet: every P is 0
    const float p = __builtin_amdgcn_exp2f(fmaf(x, sl2, -m_use));
    l_run += p;
    return p;
  };
  auto top_of = [&](const f32x16_t& x) __attribute__((always_inline)) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, x[i]);
    return top;
  };
  // P V of a tile, and the next tile's scores (K at kn, its first fragments in k) with their
  // maximum. In this order the vector instructions stand between products that they do not depend
  // on: the compiler would put a tile's products one after another, and its arithmetic behind them.
  // With two tiles a step the tile after the next has landed too, and its first fragments come
  // into k (one tree of 61 nodes over 30 thousand tokens, P in one value: 52 -> 50.5 us; V's too:
  // no faster).
  constexpr int A = KS < 4 ? KS : 4;  // fragments of K ahead
  auto add = [&](f32x16_t& sc, const char* vt, const char* kn, const char* after, uint4 (&k)[KS],
                 float& top) __attribute__((always_inline)) {
    // weights between the scores' products (the first half's at least); the others between V's
    // first
    constexpr int E = 12;
    uint4 v[2][DT];
    float x[16];
    uint32_t p[2][8];  // the weights' first parts, and the rest of them
    auto weights = [&](int from, int to) __attribute__((always_inline)) {
#pragma unroll
      for (int i = from; i < to; ++i) {
        x[i] = weight(sc[i]);
        if (i & 1) {
          // (float16's first part is cut, one instruction instead of five: the rest is exact)
          const uint32_t h =
              F16 ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x[i - 1], x[i]))
                  : pack_bf2(x[i - 1], x[i]);
          p[0][i / 2] = h;
          p[1][i / 2] = pack_e2<F16>(x[i - 1] - e2f<F16>((uint16_t)h),
                                     x[i] - e2f<F16>((uint16_t)(h >> 16)));
        }
      }
    };
    f32x16_t next;
#pragma unroll
    for (int i = 0; i < 16; ++i) next[i] = 0.f;
    values(vt, 0, v[0]);
    // ahead of the SIMD's other wave, if that is between its tiles (64 trees of 36 nodes over 5000
    // tokens, P in one value: 238 against 245 us)
    __builtin_amdgcn_s_setprio(1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      next = mfma32<F16>(k[i], qf[i], next);
      if (i + A < KS) k[i + A] = k_of(kn, i + A);
      weights(E * i / KS, E * (i + 1) / KS);
      __builtin_amdgcn_sched_barrier(0);
    }
    values(vt, 1, v[1]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < 4 * DT; ++n) {  // product j of both parts, of all dims
      const int j = n / (2 * DT), t = n % DT, m = n - 2 * DT;
      const uint32_t* const w = p[n / DT % 2] + 4 * j;
      oacc[t] = mfma32<F16>(v[j][t], make_uint4(w[0], w[1], w[2], w[3]), oacc[t]);
      if (m < 0) weights(E + (16 - E) * n / (2 * DT), E + (16 - E) * (n + 1) / (2 * DT));
      if constexpr (PT == 2) {
        if (m == 0)
#pragma unroll
          for (int i = 0; i < A; ++i) k[i] = k_of(after, i);
      }
      if (m >= 0) {
        constexpr int M = 8 / DT;
#pragma unroll
        for (int i = 0; i < M; ++i) {
          const float y = next[M * m + i];
          top = m == 0 && i == 0 ? y : fmaxf(top, y);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    sc = next;
  };
  for (int w0 = begin; w0 < end; w0 += WIN) {
    const int wend = min(end, w0 + WIN), nstep = (wend - w0 + STEP - 1) / STEP;
    if (w0 != begin) __syncthreads();  // the last window has been read
    int hole = 0;  // a missing block
    for (int i = tid; i < nstep * STEP; i += 64 * W) {
      const int64_t at = w0 + i < wend ? a.pages.row(b, w0 + i) : -1;
      rows[i] = at < 0 ? -1 : (int)at + kvh * a.pages.block_size;
      hole |= at < 0 && w0 + i < wend;
    }
    if (w0 == begin) {  // (while the block tables are on their way)
      const uint64_t all = a.parents ? ancestors(node_parent(up, lane)) : ~0ull >> (63 - lane);
      mask = (uint64_t)__shfl((long long)all, node);
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        qf[i].x ^= flip, qf[i].y ^= flip, qf[i].z ^= flip, qf[i].w ^= flip;
        // wait for q here: at its first use the compiler, which does not count the fetches, would
        // wait for all of them, in every step
        asm volatile("" : "+v"(qf[i].x), "+v"(qf[i].y), "+v"(qf[i].z), "+v"(qf[i].w));
      }
    }
    const bool holes = __syncthreads_or(hole);
#pragma unroll
    for (int s = 0; s < RING - 1; ++s)
      if (s < nstep) fetch(s);
    f32x16_t sc;  // of the tile at hand, and each lane's maximum of them
    float top;
    if (nstep >= RING - 1)
      wait_vm<(RING - 2) * LD>();  // step 0 has landed
    else
      wait_vm<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    sc = scores(0, 0);
    top = top_of(sc);
    uint4 k[KS];
    if constexpr (PT == 2)
#pragma unroll
      for (int i = 0; i < A; ++i) k[i] = k_of(lds + part * PART_B + TILE_B, i);
#pragma unroll 1
    for (int s = 0; s < nstep; ++s) {
      if (nstep - 1 - s >= RING - 2)
        wait_vm<(RING - 3) * LD>();  // step s + 1 has landed
      else
        wait_vm<0>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      // The slot filled now was read a step ago: every wave is past that.
      if (s + RING - 1 < nstep) fetch(s + RING - 1);
      const int t0 = w0 + s * STEP;
      const bool masked = t0 + STEP > c.context || holes;
      if (masked) clean(s, t0);
      if (row0 >= R) continue;
#pragma unroll
      for (int q = 0; q < PT; ++q) {
        auto tile = [&](int ahead) {  // (behind the last: of nothing)
          const int st = s + (q + ahead) / PT;
          return lds + (st % RING) * STEP_B + part * PART_B + (q + ahead) % PT * TILE_B;
        };
        const char* const kn = tile(1);
        if constexpr (PT == 1) {
#pragma unroll
          for (int i = 0; i < A; ++i) k[i] = k_of(kn, i);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (masked) {
          const int at = PTOK * part + 32 * q;
          const uint32_t here = (uint32_t)__ballot(rows[s * STEP + at + ln] >= 0);
          // of the tile's tokens from `past` on not every row attends each
          const int past = max(c.context - t0 - at, 0);
          const uint64_t tree = past ? mask << min(past, 63) : mask >> min(t0 + at - c.context, 63);
          const uint32_t on = here & (past >= 32 ? ~0u : (uint32_t)tree | ((1u << past) - 1));
#pragma unroll
          for (int i = 0; i < 16; ++i)
            sc[i] = on >> (4 * lh) >> (8 * (i >> 2) + (i & 3)) & 1 ? sc[i] : -INFINITY;
          top = top_of(sc);
        }
        rescale(pair32_max(top) * sl2);
        add(sc, tile(0) + HALF_B, kn, tile(2), k, top);
      }
    }
  }
  l_run = pair32_sum(l_run);

  // The other parts' waves hand (max, sum, O) to the first part's: XCH values per lane.
  if constexpr (TW > 1) {
    __syncthreads();  // every wave is past its last read of the ring
    float* const x = reinterpret_cast<float*>(lds) + (size_t)(wave % RW) * XCH * 64 + lane;
    constexpr int XP = RW * XCH * 64;  // values of a part
    if (part > 0) {
      float* const w = x + (size_t)(part - 1) * XP;
      w[0] = m_run;
      w[64] = l_run;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) w[64 * (2 + 16 * t + i)] = oacc[t][i];
    }
    __syncthreads();
    if (part > 0) return;
    float m = m_run;
#pragma unroll
    for (int p = 1; p < TW; ++p) m = fmaxf(m, x[(p - 1) * XP]);
    const float m_use = m == -INFINITY ? 0.f : m;
    const float f0 = __builtin_amdgcn_exp2f(m_run - m_use);
    l_run *= f0;
#pragma unroll
    for (int t = 0; t < DT; ++t) oacc[t] *= f0;
#pragma unroll
    for (int p = 1; p < TW; ++p) {
      const float* const w = x + (size_t)(p - 1) * XP;
      const float fp = __builtin_amdgcn_exp2f(w[0] - m_use);
      l_run += fp * w[64];
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) oacc[t][i] += fp * w[64 * (2 + 16 * t + i)];
    }
    m_run = m;
  }
  // A value of V that is not finite: it was taken out, or the two parts of its weights made NaN of
  // it. Such values' sum, of its row's attended tokens, takes the place of the dim's.
  float finite = 0.f;  // (0 of finite sums, else NaN)
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) finite = fmaf(oacc[t][i], 0.f, finite);
  const bool whole = __ballot(finite != 0.f && l_run == l_run) != 0;  // else among the nodes only
  if (__builtin_expect(odd || whole, 0)) {
    f32x16_t e[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) e[t][i] = 0.f;
#pragma unroll 1
    for (int k = whole ? begin : max(begin, c.context); k < end; ++k) {
      const int64_t r = a.pages.row(b, k);
      if (r < 0) continue;
      const bool mine = k < c.context || ((mask >> (k - c.context)) & 1);
      const uint16_t* const d = a.vc + (r + (int64_t)kvh * a.pages.block_size) * D + 4 * lh;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint2 x = *reinterpret_cast<const uint2*>(d + 32 * t + 8 * i);
          const uint32_t w[2] = {x.x & inf_halves<F16>(x.x), x.y & inf_halves<F16>(x.y)};
#pragma unroll
          for (int n = 0; n < 4; ++n)
            e[t][4 * i + n] += mine ? e2f<F16>((uint16_t)(w[n / 2] >> (n & 1) * 16)) : 0.f;
        }
    }
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) oacc[t][i] = e[t][i] == 0.f ? oacc[t][i] : e[t][i];
  }
  if (row >= R) return;
  if (c.splits <= 1) {
    const float inv = node < c.nodes && l_run != 0.f ? 1.f / l_run : 0.f;
    uint16_t* const o = a.out + (((int64_t)b * a.T + node) * a.Hq + head) * D + 8 * lh;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 16; i += 8) {
        // 4 dims of 8 each: the halves of the wave exchange them for 8 that are neighbours
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[e] = inv == 0.f ? 0u
                            : pack_e2<F16>(oacc[t][i + 2 * e] * inv, oacc[t][i + 2 * e + 1] * inv);
        const auto x = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
        const auto y = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
        *reinterpret_cast<uint4*>(o + 32 * t + 2 * i) = make_uint4(x[0], y[0], x[1], y[1]);
      }
    return;
  }
  const int64_t at = ((int64_t)pair * f.splits + split) * f.RP + row;
  float* const o = f.ws_o + at * D + 4 * lh;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      *reinterpret_cast<float4*>(o + 32 * t + 2 * i) =
          make_float4(oacc[t][i], oacc[t][i + 1], oacc[t][i + 2], oacc[t][i + 3]);
  if (lh == 0) *reinterpret_cast<float2*>(f.ws_ml + 2 * at) = make_float2(m_run, l_run);
}

// Joins the splits of a row: D / 4 lanes per row, where there are two splits or more.
constexpr int JT = 256;
template <bool F16, int D>
__global__ void __launch_bounds__(JT) tree_attn_join_kernel(FastArgs f, int step) {
  constexpr int L = D / 4, RPB = JT / L;
  const TreeArgs& a = f.t;
  const int Hkv = a.pages.Hkv, G = a.Hq / Hkv, R = a.T * G;
  const int pair = blockIdx.y, b = pair / Hkv, kvh = pair - b * Hkv;
  const Cut c = cut_of(a, a.cl[b], a.counts ? a.counts[b] : a.T, f.splits, step);
  if (c.splits <= 1) return;
  const int row = blockIdx.x * RPB + threadIdx.x / L, l = threadIdx.x % L;
  if (row >= R) return;
  const int node = row / G, head = kvh * G + row - node * G;
  const int64_t at = (int64_t)pair * f.splits * f.RP + row;
  const float2* const ml = reinterpret_cast<const float2*>(f.ws_ml) + at;
  const float4* const o = reinterpret_cast<const float4*>(f.ws_o) + at * L + l;
  // A lane has every L-th split's weight, and four dims of all.
  constexpr int N = MAX_SPLITS / L, AT_ONCE = 8;
  float2 w[N];
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int z = i * L + l;
    w[i] = z < c.splits ? ml[(int64_t)z * f.RP] : make_float2(-INFINITY, 0.f);
    m = fmaxf(m, w[i].x);
  }
#pragma unroll
  for (int x = L / 2; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
  const float m_use = m == -INFINITY ? 0.f : m;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float mine = __builtin_amdgcn_exp2f(w[i].x - m_use);
    sum += mine * w[i].y;
#pragma unroll
    for (int z0 = i * L; z0 < (i + 1) * L; z0 += AT_ONCE) {
      if (z0 >= c.splits) break;
      float4 v[AT_ONCE];
#pragma unroll
      for (int z = 0; z < AT_ONCE; ++z)
        if (z0 + z < c.splits) v[z] = o[(int64_t)(z0 + z) * f.RP * L];
#pragma unroll
      for (int z = 0; z < AT_ONCE; ++z) {
        if (z0 + z >= c.splits) break;
        const float x = __shfl(mine, (threadIdx.x & 63 & ~(L - 1)) + z0 % L + z);
        acc.x += x * v[z].x, acc.y += x * v[z].y, acc.z += x * v[z].z, acc.w += x * v[z].w;
      }
    }
  }
#pragma unroll
  for (int x = L / 2; x; x >>= 1) sum += __shfl_xor(sum, x);
  const float inv = node < c.nodes && sum != 0.f ? 1.f / sum : 0.f;
  uint2 y =
      make_uint2(pack_e2<F16>(acc.x * inv, acc.y * inv), pack_e2<F16>(acc.z * inv, acc.w * inv));
  if (inv == 0.f) y = make_uint2(0u, 0u);
  *reinterpret_cast<uint2*>(a.out + (((int64_t)b * a.T + node) * a.Hq + head) * D + 4 * l) = y;
}

struct Plan {
  int rw;          // waves side by side on rows; 8 / rw on tokens
  int rb, splits;  // blocks of 32 rw rows, parts of a sequence's tokens
  size_t values;   // rows of the workspace
};
Plan plan_of(int B, int T, int Hq, int Hkv, int D) {
  const int R = T * (Hq / Hkv);
  Plan p;
  // The fewest waves on rows that hold them, of 4 and 8: 64 trees over 2500 tokens, 4 KV heads of
  // 128 dims, 28 rows, 88 us with 4 and 92 with 8, 112 rows 102 and 105, 224 rows 192 and 152; of 2
  // where a token is 128 bytes: 28 rows of 64 dims 45 us with 2, 62 with 4 and 68 with 8, 56 rows
  // 48, 65 and 71, 112 rows 84, 71 and 74.
  p.rw = R <= 64 && D == 64 ? 2 : (R <= 128 ? 4 : 8);
  p.rb = (int)cdiv(R, 32 * p.rw);
  const int64_t groups = (int64_t)B * Hkv * p.rb;
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(MAX_SPLITS, 256 / groups));
  p.values = p.splits > 1 ? (size_t)B * Hkv * p.splits * p.rb * 32 * p.rw : 0;
  return p;
}
bool fast_dim(int D) { return D == 64 || D == 128; }

template <bool F16, int D, int RW>
int go(const FastArgs& a, const Plan& p, hipStream_t st) {
  constexpr int LDS = RING * step_of<RW>() / 32 * 2 * TILE<D> + WIN * 4;
  constexpr auto kern = tree_attn_kernel<F16, D, RW>;
  if (int rc = allow_dynamic_lds<kern, LDS>()) return rc;
  // Blocks of rows that read the same tokens run on one XCD: their ids are equal modulo 8.
  int64_t x = (int64_t)a.t.B * a.t.pages.Hkv * p.splits;
  if (p.rb > 1) x = cdiv(x, 8) * 8;
  kern<<<dim3((unsigned)x, (unsigned)p.rb), 512, LDS, st>>>(a);
  if (p.splits > 1) {
    const int R = a.t.T * (a.t.Hq / a.t.pages.Hkv);
    tree_attn_join_kernel<F16, D><<<dim3((unsigned)cdiv(R, JT / (D / 4)),
                                         (unsigned)(a.t.B * a.t.pages.Hkv)), JT, 0, st>>>(
        a, step_of<RW>());
  }
  return launch_check("paged_tree_attn");
}
template <bool F16, int D>
int go_form(const FastArgs& a, const Plan& p, hipStream_t st) {
  if constexpr (D == 64)
    if (p.rw == 2) return go<F16, D, 2>(a, p, st);
  return p.rw == 4 ? go<F16, D, 4>(a, p, st) : go<F16, D, 8>(a, p, st);
}

}  // namespace

extern "C" size_t grpo_paged_tree_attn_workspace_bytes(int B, int T, int Hq, int Hkv, int D) {
  if (B < 1 || T < 1 || T > TREE_MAX || Hkv < 1 || Hq < 1 || Hq % Hkv || !fast_dim(D)) return 0;
  return plan_of(B, T, Hq, Hkv, D).values * (D + 2) * sizeof(float);
}

extern "C" int grpo_paged_tree_attn(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh,
                                    int f16, const void* k_cache, const void* v_cache,
                                    int64_t num_blocks, const int32_t* block_tables,
                                    int64_t bt_stride, int block_size, int max_blocks,
                                    const int32_t* context_lens, const int32_t* parents,
                                    int64_t parents_stride, const int32_t* counts, float scale,
                                    void* out, int B, int T, int Hq, int Hkv, int D,
                                    void* workspace, size_t workspace_bytes,
                                    grpo_stream_t stream) {
  if (B < 0 || T < 1 || num_blocks < 1 || block_size < 1 || max_blocks < 1 || Hq < 1 || Hkv < 1 ||
      Hq % Hkv || D < 1 || (int64_t)max_blocks * block_size >= (1ll << 31))
    return einval("bad attention dimensions");
  if (T > TREE_MAX) return einval("a drafted tree has at most 64 nodes");
  if (D > GD) return einval("head_dim at most 512");
  if (!std::isfinite(scale)) return einval("the scale must be finite");
  // (the plain kernel: 256 threads for each node, fewer than 2^32 in a row of its grid)
  if (Hq > 65535 || (int64_t)B * T >= (1ll << 24))
    return einval("at most 65535 heads and 2^24 - 1 nodes");
  if (B == 0) return GRPO_OK;
  if (!q || !k_cache || !v_cache || !block_tables || !context_lens || !out)
    return einval("null pointer");
  const TreeArgs a{static_cast<const uint16_t*>(q),
                   q_sb,
                   q_st,
                   q_sh,
                   static_cast<const uint16_t*>(k_cache),
                   static_cast<const uint16_t*>(v_cache),
                   {block_tables, bt_stride, num_blocks, block_size, max_blocks, Hkv},
                   context_lens,
                   parents,
                   parents_stride,
                   counts,
                   static_cast<uint16_t*>(out),
                   B,
                   T,
                   Hq,
                   D,
                   scale};
  hipStream_t st = as_stream(stream);
  if (fast_dim(D) && ((q_sb | q_st | q_sh) & 7) == 0 && aligned16(q) && aligned16(k_cache) &&
      aligned16(v_cache) && aligned16(out) && (int64_t)B * Hkv < 65536 &&
      num_blocks * Hkv * block_size < (1ll << 31) &&
      (int64_t)max_blocks * block_size <= (1ll << 31) - 2 * WIN) {
    const Plan p = plan_of(B, T, Hq, Hkv, D);
    const size_t need = p.values * (D + 2) * sizeof(float);
    if (need && (!workspace || !aligned16(workspace) || workspace_bytes < need)) {
      set_error("tree attention workspace: %zu bytes, 16-byte aligned", need);
      return GRPO_EWORKSPACE;
    }
    float* const ws = static_cast<float*>(workspace);
    const FastArgs f{a, p.splits, p.rb * 32 * p.rw, ws, ws + p.values * D};
    if (f16) return D == 64 ? go_form<true, 64>(f, p, st) : go_form<true, 128>(f, p, st);
    return D == 64 ? go_form<false, 64>(f, p, st) : go_form<false, 128>(f, p, st);
  }
  const dim3 grid((unsigned)(B * T), (unsigned)Hq);
  if (f16)
    tree_attn_plain_kernel<true><<<grid, GT, 0, st>>>(a);
  else
    tree_attn_plain_kernel<false><<<grid, GT, 0, st>>>(a);
  return launch_check("paged_tree_attn");
}

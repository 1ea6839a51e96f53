// The cache side of checking a tree of drafted tokens (gfx950): rotating and storing the
// nodes' queries, keys and values (grpo_paged_rope_append), and keeping the nodes that the
// sampled tokens accept (grpo_draft_tree_accept).
//
// The append is the reference's fused_qkv_rope + KV update (src/triton_kernels/fused_ops.py:
// 198-219, paged_kv.py:253-319) for several tokens per sequence; the rotation is float32 from
// 16-bit or float32 tables and rounds once.
#include "tree.hpp"

using namespace grpo;

namespace {

constexpr int RT = 256;  // threads

struct Strided {
  const uint16_t* p;
  int64_t b, t, h;  // strides in values
  __device__ __forceinline__ const uint16_t* at(int bi, int ti, int hi) const {
    return p + (int64_t)bi * b + (int64_t)ti * t + (int64_t)hi * h;
  }
};

struct AppendArgs {
  Strided q, k, v;
  const void* cos;
  const void* sin;
  int max_pos;
  const int32_t* pos;  // or null: context + node
  int64_t pos_stride;
  const int32_t* cl;
  const int32_t* counts;
  uint16_t* q_out;  // [B][T][Hq][D]
  uint16_t* kc;
  uint16_t* vc;
  Pages pages;
  int B, T, Hq, D;
};

// N values of a 16-bit row, or of a table, as floats.
template <bool F16, int N>
__device__ __forceinline__ void load_n(const uint16_t* p, float (&o)[N]) {
  if constexpr (N == 8) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[2 * i] = e2f<F16>((uint16_t)w[i]);
      o[2 * i + 1] = e2f<F16>((uint16_t)(w[i] >> 16));
    }
  } else {
    o[0] = e2f<F16>(p[0]);
  }
}
template <bool F16, bool TF32, int N>
__device__ __forceinline__ void load_table(const void* t, int64_t at, float (&o)[N]) {
  if constexpr (!TF32) {
    load_n<F16, N>(static_cast<const uint16_t*>(t) + at, o);
  } else {
    const float* const f = static_cast<const float*>(t) + at;
    if constexpr (N == 8) {
      const float4 a = *reinterpret_cast<const float4*>(f);
      const float4 b = *reinterpret_cast<const float4*>(f + 4);
      o[0] = a.x, o[1] = a.y, o[2] = a.z, o[3] = a.w;
      o[4] = b.x, o[5] = b.y, o[6] = b.z, o[7] = b.w;
    } else {
      o[0] = f[0];
    }
  }
}
template <bool F16, int N>
__device__ __forceinline__ void store_n(uint16_t* p, const float (&o)[N]) {
  if constexpr (N == 8)
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_e2<F16>(o[0], o[1]), pack_e2<F16>(o[2], o[3]),
                                              pack_e2<F16>(o[4], o[5]), pack_e2<F16>(o[6], o[7]));
  else
    p[0] = f2e<F16>(o[0]);
}
template <int N>
__device__ __forceinline__ void copy_n(uint16_t* to, const uint16_t* from) {
  if constexpr (N == 8)
    *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
  else
    to[0] = from[0];
}

// A workgroup per node row: a thread takes N pairs (d, d + D/2) of one head, then N values of
// v. N = 8, 16 bytes a load, where the addresses allow it. Bound by HBM where there are many rows:
// 8 x 2048 tokens of 28 and 4 heads of 128, 302 MB read and written in 54 us (5.6 TB/s); 32 x 61
// of them 9 us (27 MB), 8 x 4 of 12 and 2 heads 3.8 us, the launch.
template <bool F16, bool TF32, int N>
__global__ void __launch_bounds__(RT) rope_append_rows_kernel(AppendArgs a) {
  const int b = blockIdx.x / a.T, t = blockIdx.x - b * a.T;
  const int context = a.cl[b], half = a.D / 2, per = half / N, Hkv = a.pages.Hkv;
  const bool used = t < nodes_of(a.counts, b, a.T, context);
  uint16_t* const qo = a.q_out + (int64_t)blockIdx.x * a.Hq * a.D;
  if (!used) {
    const float zero[N] = {};
    for (int i = threadIdx.x; i < a.Hq * 2 * per; i += RT) store_n<F16, N>(qo + N * i, zero);
    return;
  }
  const int64_t pos = a.pos ? a.pos[(int64_t)b * a.pos_stride + t] : (int64_t)context + t;
  const int64_t tab = (pos < 0 ? 0 : (pos >= a.max_pos ? a.max_pos - 1 : pos)) * a.D;
  const int64_t row = a.pages.row(b, (int64_t)context + t);
  for (int i = threadIdx.x; i < (a.Hq + Hkv) * per; i += RT) {
    const int h = i / per, d = N * (i - h * per);
    const bool is_q = h < a.Hq;
    if (!is_q && row < 0) continue;
    const uint16_t* const x = (is_q ? a.q.at(b, t, h) : a.k.at(b, t, h - a.Hq)) + d;
    float x1[N], x2[N], c1[N], c2[N], s1[N], s2[N];
    load_n<F16, N>(x, x1);
    load_n<F16, N>(x + half, x2);
    load_table<F16, TF32, N>(a.cos, tab + d, c1);
    load_table<F16, TF32, N>(a.cos, tab + d + half, c2);
    load_table<F16, TF32, N>(a.sin, tab + d, s1);
    load_table<F16, TF32, N>(a.sin, tab + d + half, s2);
    float lo[N], hi[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      lo[e] = x1[e] * c1[e] - x2[e] * s1[e];
      hi[e] = x2[e] * c2[e] + x1[e] * s2[e];
    }
    uint16_t* const o =
        (is_q ? qo + (int64_t)h * a.D
              : a.kc + (row + (int64_t)(h - a.Hq) * a.pages.block_size) * a.D) + d;
    store_n<F16, N>(o, lo);
    store_n<F16, N>(o + half, hi);
  }
  if (row < 0) return;
  for (int i = threadIdx.x; i < Hkv * 2 * per; i += RT) {
    const int h = i / (2 * per), d = N * (i - h * 2 * per);
    copy_n<N>(a.vc + (row + (int64_t)h * a.pages.block_size) * a.D + d, a.v.at(b, t, h) + d);
  }
}

struct AcceptArgs {
  const int64_t* drafted;
  const int64_t* sampled;
  const int32_t* parents;
  int64_t ds, ss, ps;  // row strides
  const int32_t* cl;
  const int32_t* counts;
  uint16_t* kc;  // [layers][num_blocks][Hkv][block_size][D]
  uint16_t* vc;
  int64_t layer_rows;  // rows of D values per layer
  Pages pages;
  int layers, B, T, D;
  int64_t eos, pad;
  int64_t* tokens;  // [B][T]
  int32_t* accepted;
  int32_t* path;
};

// Every wave walks the tree by itself (a node per lane): at node cur the sampled token is looked
// for among cur's children, the lowest first. Children come after their parent, so the walk
// takes at most T steps and the node at depth j moves from a slot >= j: its new slot has been
// read before it is written, in one thread's program order. A thread moves N values of one
// (layer, K or V, head). 8 trees of 7 nodes, 28 layers of 2 heads of 128: 4.2 us; 64 of 61 with 4
// heads 8.8 us (20 MB moved).
template <int N>
__global__ void __launch_bounds__(RT) tree_accept_kernel(AcceptArgs a) {
  const int b = blockIdx.y, lane = threadIdx.x & 63;
  const int context = a.cl[b], n = nodes_of(a.counts, b, a.T, context);
  int64_t want = 0, has = 0;
  int up = -1, mine = -1;
  if (lane < n) {
    has = a.drafted[(int64_t)b * a.ds + lane];
    want = a.sampled[(int64_t)b * a.ss + lane];
    up = node_parent(a.parents[(int64_t)b * a.ps + lane], lane);
  }
  int len = 0;
  for (int cur = n > 0 ? 0 : -1; cur >= 0;) {
    if (lane == len) mine = cur;  // the node at this depth
    ++len;
    const uint32_t w0 = __builtin_amdgcn_readlane((int)(uint32_t)want, cur);
    const uint32_t w1 = __builtin_amdgcn_readlane((int)(uint32_t)(want >> 32), cur);
    const int64_t token = (int64_t)((uint64_t)w1 << 32 | w0);
    const uint64_t child = __ballot(lane < n && up == cur && has == token);
    cur = child && token >= 0 && token != a.eos ? __builtin_ctzll(child) : -1;
  }
  if (blockIdx.x == 0 && threadIdx.x < (unsigned)a.T) {
    const int64_t at = (int64_t)b * a.T + lane;
    a.tokens[at] = lane < len ? a.sampled[(int64_t)b * a.ss + mine] : a.pad;
    a.path[at] = lane < len ? mine : -1;
    if (lane == 0) a.accepted[b] = len;
  }
  // Rows of the moved nodes, -1 where there is nothing to move.
  const bool moves = lane < len && mine != lane;
  const int64_t src = moves ? a.pages.row(b, (int64_t)context + mine) : -1;
  const int64_t dst = src >= 0 ? a.pages.row(b, (int64_t)context + lane) : -1;
  if (!__ballot(dst >= 0)) return;
  const int per = a.D / N, Hkv = a.pages.Hkv;
  const int i = blockIdx.x * RT + threadIdx.x;
  const int unit = i / per, d = N * (i - unit * per);
  const bool on = unit < a.layers * Hkv * 2;
  const int l = unit / (2 * Hkv), h = unit / 2 - l * Hkv;
  uint16_t* const base = ((unit & 1) ? a.vc : a.kc) +
                         (on ? (l * a.layer_rows + (int64_t)h * a.pages.block_size) * a.D + d : 0);
  for (int j = 1; j < len; ++j) {
    const int64_t to = __shfl((long long)dst, j), from = __shfl((long long)src, j);
    if (on && to >= 0) copy_n<N>(base + to * a.D, base + from * a.D);
  }
}

bool pages_ok(int64_t num_blocks, int block_size, int max_blocks, int Hq, int Hkv, int D) {
  return num_blocks > 0 && block_size > 0 && max_blocks > 0 && Hq > 0 && Hkv > 0 &&
         Hq % Hkv == 0 && D > 0 && (int64_t)max_blocks * block_size < (1ll << 31);
}

template <bool F16, bool TF32>
int append(const AppendArgs& a, bool vec, hipStream_t st) {
  const unsigned grid = (unsigned)(a.B * a.T);
  if (vec)
    rope_append_rows_kernel<F16, TF32, 8><<<grid, RT, 0, st>>>(a);
  else
    rope_append_rows_kernel<F16, TF32, 1><<<grid, RT, 0, st>>>(a);
  return launch_check("paged_rope_append");
}

}  // namespace

extern "C" int grpo_paged_rope_append(
    const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb,
    int64_t k_st, int64_t k_sh, const void* v, int64_t v_sb, int64_t v_st, int64_t v_sh, int f16,
    const void* cos_table, const void* sin_table, int table_f32, int max_pos,
    const int32_t* positions, int64_t pos_stride, const int32_t* context_lens,
    const int32_t* counts, void* q_out, void* k_cache, void* v_cache, int64_t num_blocks,
    const int32_t* block_tables, int64_t bt_stride, int block_size, int max_blocks, int B, int T,
    int Hq, int Hkv, int D, grpo_stream_t stream) {
  if (B < 0 || T < 0 || D % 2 || max_pos <= 0 ||
      !pages_ok(num_blocks, block_size, max_blocks, Hq, Hkv, D))
    return einval("bad rope/append dimensions");
  // (256 threads for each row, fewer than 2^32 in a launch)
  if ((int64_t)B * T >= (1ll << 24)) return einval("at most 2^24 - 1 tokens");
  if (B == 0 || T == 0) return GRPO_OK;
  if (!q || !k || !v || !cos_table || !sin_table || !context_lens || !q_out || !k_cache ||
      !v_cache || !block_tables)
    return einval("null pointer");
  const AppendArgs a{{static_cast<const uint16_t*>(q), q_sb, q_st, q_sh},
                     {static_cast<const uint16_t*>(k), k_sb, k_st, k_sh},
                     {static_cast<const uint16_t*>(v), v_sb, v_st, v_sh},
                     cos_table,
                     sin_table,
                     max_pos,
                     positions,
                     pos_stride,
                     context_lens,
                     counts,
                     static_cast<uint16_t*>(q_out),
                     static_cast<uint16_t*>(k_cache),
                     static_cast<uint16_t*>(v_cache),
                     {block_tables, bt_stride, num_blocks, block_size, max_blocks, Hkv},
                     B,
                     T,
                     Hq,
                     D};
  const int64_t strides = q_sb | q_st | q_sh | k_sb | k_st | k_sh | v_sb | v_st | v_sh;
  const bool vec = D % 16 == 0 && strides % 8 == 0 && aligned16(q) && aligned16(k) &&
                   aligned16(v) && aligned16(cos_table) && aligned16(sin_table) &&
                   aligned16(q_out) && aligned16(k_cache) && aligned16(v_cache);
  hipStream_t st = as_stream(stream);
  if (f16) return table_f32 ? append<true, true>(a, vec, st) : append<true, false>(a, vec, st);
  return table_f32 ? append<false, true>(a, vec, st) : append<false, false>(a, vec, st);
}

extern "C" int grpo_draft_tree_accept(
    const int64_t* drafted, int64_t drafted_stride, const int32_t* parents, int64_t parents_stride,
    const int64_t* sampled, int64_t sampled_stride, const int32_t* context_lens,
    const int32_t* counts, void* k_cache, void* v_cache, int layers, int64_t num_blocks,
    const int32_t* block_tables, int64_t bt_stride, int block_size, int max_blocks, int B, int T,
    int Hkv, int D, int64_t eos, int64_t pad, int64_t* tokens, int32_t* accepted, int32_t* path,
    grpo_stream_t stream) {
  if (B < 0 || T < 1 || layers < 1 || !pages_ok(num_blocks, block_size, max_blocks, Hkv, Hkv, D))
    return einval("bad dimensions of the drafted tree or the cache");
  if (T > TREE_MAX) return einval("a drafted tree has at most 64 nodes");
  if (B > 65535) return einval("at most 65535 sequences");
  if (B == 0) return GRPO_OK;
  if (!drafted || !parents || !sampled || !context_lens || !k_cache || !v_cache ||
      !block_tables || !tokens || !accepted || !path)
    return einval("null pointer");
  const AcceptArgs a{drafted,
                     sampled,
                     parents,
                     drafted_stride,
                     sampled_stride,
                     parents_stride,
                     context_lens,
                     counts,
                     static_cast<uint16_t*>(k_cache),
                     static_cast<uint16_t*>(v_cache),
                     num_blocks * Hkv * block_size,
                     {block_tables, bt_stride, num_blocks, block_size, max_blocks, Hkv},
                     layers,
                     B,
                     T,
                     D,
                     eos,
                     pad,
                     tokens,
                     accepted,
                     path};
  const bool vec = D % 8 == 0 && aligned16(k_cache) && aligned16(v_cache);
  const int64_t threads = (int64_t)layers * Hkv * 2 * (D / (vec ? 8 : 1));
  if (threads >= (1ll << 31)) return einval("too many layers and heads");
  const dim3 grid((unsigned)cdiv(threads, RT), (unsigned)B);
  hipStream_t st = as_stream(stream);
  if (vec)
    tree_accept_kernel<8><<<grid, RT, 0, st>>>(a);
  else
    tree_accept_kernel<1><<<grid, RT, 0, st>>>(a);
  return launch_check("draft_tree_accept");
}

// Paged GQA attention of a tree of drafted tokens (grpo_paged_tree_attn), gfx950: T nodes per
// sequence whose keys and values stand in the cache's slots after its context_lens[b] tokens;
// node i attends those tokens, its ancestors and itself. What the reference's decode attention
// (src/triton_kernels/paged_kv.py:63-251) does for one token, for a tree of them.
//
// A token that a node does not attend is not read for it: whatever stands there (NaN of a slot
// never written, another branch) stays out. A node that attends nothing gets 0.
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
  const int64_t last = used ? (int64_t)context + t + 1 : 0;
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

}  // namespace

extern "C" size_t grpo_paged_tree_attn_workspace_bytes(int B, int T, int Hq, int Hkv, int D) {
  (void)B, (void)T, (void)Hq, (void)Hkv, (void)D;
  return 0;
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
  if (Hq > 65535 || (int64_t)B * T >= (1ll << 31)) return einval("too many rows or heads");
  if (B == 0) return GRPO_OK;
  if (!q || !k_cache || !v_cache || !block_tables || !context_lens || !out)
    return einval("null pointer");
  (void)workspace, (void)workspace_bytes;
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
  const dim3 grid((unsigned)(B * T), (unsigned)Hq);
  if (f16)
    tree_attn_plain_kernel<true><<<grid, GT, 0, as_stream(stream)>>>(a);
  else
    tree_attn_plain_kernel<false><<<grid, GT, 0, as_stream(stream)>>>(a);
  return launch_check("paged_tree_attn");
}

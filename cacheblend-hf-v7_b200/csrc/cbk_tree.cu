// Attention of a tree of drafted tokens over the cache.
//
// Node i of T nodes sees cache rows [0, n_ctx) and, of the rows n_ctx + j that
// hold the nodes' own K and V, those whose bit j is set in words[i]:
//   out[i][h] = softmax_t(scale q[i][h] . k[t][h / G]) . v[t][h / G].
// n_ctx is read on the device, so a captured step stays valid as it advances.
//
// One CTA per (node, q head), a warp per key, an online softmax per warp and a
// merge of the warps: every key row is read once per query row.
#include "cbk_common.cuh"

namespace cbk {

constexpr int kTreeThreads = 128;
constexpr int kTreeWarps = kTreeThreads / 32;

template <int DT, int HD>
__global__ void __launch_bounds__(kTreeThreads)
tree_attn_kernel(const uint16_t* __restrict__ q, const uint16_t* __restrict__ kc, const uint16_t* __restrict__ vc,
                 int64_t kv_stride, const int64_t* __restrict__ n_ctx_ptr, const uint32_t* __restrict__ words,
                 int64_t words_stride, int n_nodes, int64_t cap, int n_q, int group, float scale_log2,
                 uint16_t* __restrict__ out, int32_t* status) {
  using E = Elem<DT>;
  constexpr int kD = HD / 32;
  __shared__ float s_m[kTreeWarps], s_l[kTreeWarps], s_o[kTreeWarps][HD];
  const int node = blockIdx.x, hq = blockIdx.y, h = hq / group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n_ctx = *n_ctx_ptr;
  if (n_ctx < 0 || n_ctx + n_nodes > cap) {
    if (threadIdx.x == 0 && node == 0 && hq == 0) report(status, CBK_STATUS_BAD_INDEX);
    return;
  }
  float qf[kD], o[kD], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int d = 0; d < kD; ++d) {
    qf[d] = E::to_f(q[(static_cast<int64_t>(node) * n_q + hq) * HD + lane * kD + d]);
    o[d] = 0.f;
  }
  for (int64_t t = warp; t < n_ctx + n_nodes; t += kTreeWarps) {
    if (t >= n_ctx) {
      const int j = static_cast<int>(t - n_ctx);
      if (!((words[node * words_stride + j / 32] >> (j % 32)) & 1u)) continue;
    }
    const uint16_t* kr = kc + t * kv_stride + static_cast<int64_t>(h) * HD + lane * kD;
    const uint16_t* vr = vc + t * kv_stride + static_cast<int64_t>(h) * HD + lane * kD;
    float s = 0.f;
#pragma unroll
    for (int d = 0; d < kD; ++d) s = fmaf(qf[d], E::to_f(kr[d]), s);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= scale_log2;
    const float m_new = fmaxf(m, s);
    const float a = m == m_new ? 1.f : ex2(m - m_new), w = ex2(s - m_new);
    l = l * a + w;
    m = m_new;
#pragma unroll
    for (int d = 0; d < kD; ++d) o[d] = fmaf(w, E::to_f(vr[d]), o[d] * a);
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int d = 0; d < kD; ++d) s_o[warp][lane * kD + d] = o[d];
  __syncthreads();
  for (int d = threadIdx.x; d < HD; d += kTreeThreads) {
    float M = -INFINITY, L = 0.f, acc = 0.f;
    for (int w = 0; w < kTreeWarps; ++w)
      if (s_l[w] != 0.f) M = fmaxf(M, s_m[w]);
    for (int w = 0; w < kTreeWarps; ++w)
      if (s_l[w] != 0.f) {
        const float wt = ex2(s_m[w] - M);
        L += wt * s_l[w];
        acc += wt * s_o[w][d];
      }
    out[(static_cast<int64_t>(node) * n_q + hq) * HD + d] = E::from_f(L == 0.f ? 0.f : acc / L);
  }
}

}  // namespace cbk

using namespace cbk;

constexpr int kTreeMaxNodes = 1024;

static int check_tree_geometry(const char* who, int n_nodes, int64_t cap, int n_q_heads, int n_kv_heads,
                               int head_dim) {
  if (head_dim != 64 && head_dim != 128)
    return set_error(CBK_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128 only)", who, head_dim);
  if (n_kv_heads <= 0 || n_q_heads <= 0 || n_q_heads % n_kv_heads != 0 || n_q_heads > 4096)
    return set_error(CBK_ERR_INVALID, "%s: n_q_heads must be a multiple of n_kv_heads", who);
  if (n_nodes < 0 || n_nodes > kTreeMaxNodes)
    return set_error(CBK_ERR_UNSUPPORTED, "%s: %d nodes (at most %d)", who, n_nodes, kTreeMaxNodes);
  if (cap < n_nodes || cap > (int64_t{1} << 30))
    return set_error(CBK_ERR_INVALID, "%s: a cache of %lld rows for %d nodes", who, (long long)cap, n_nodes);
  return CBK_OK;
}

extern "C" size_t cbk_tree_attn_workspace_bytes(int n_nodes, int64_t cap, int n_q_heads, int n_kv_heads,
                                                int head_dim) {
  if (check_tree_geometry("cbk_tree_attn_workspace_bytes", n_nodes, cap, n_q_heads, n_kv_heads, head_dim) != CBK_OK)
    return 0;
  return 256;
}

extern "C" int cbk_tree_attn(const void* q, const void* k_cache, const void* v_cache, int64_t kv_row_stride,
                             const int64_t* n_ctx, const int32_t* words, int64_t words_stride, int n_nodes,
                             int64_t cap, int n_q_heads, int n_kv_heads, int head_dim, float scale, int dtype,
                             void* out, void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  if (dtype != CBK_BF16 && dtype != CBK_F16)
    return set_error(CBK_ERR_UNSUPPORTED, "cbk_tree_attn: dtype %d not supported", dtype);
  if (int rc = check_tree_geometry("cbk_tree_attn", n_nodes, cap, n_q_heads, n_kv_heads, head_dim)) return rc;
  if (n_nodes == 0) return CBK_OK;
  if (kv_row_stride < static_cast<int64_t>(n_kv_heads) * head_dim || kv_row_stride % 8 != 0 ||
      words_stride < (n_nodes + 31) / 32)
    return set_error(CBK_ERR_INVALID, "cbk_tree_attn: bad strides (cache %lld, words %lld)", (long long)kv_row_stride,
                     (long long)words_stride);
  if (!q || !k_cache || !v_cache || !n_ctx || !words || !out || !workspace)
    return set_error(CBK_ERR_INVALID, "cbk_tree_attn: null pointer argument");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
       reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15u)
    return set_error(CBK_ERR_INVALID, "cbk_tree_attn: q, caches, out and workspace must be 16-byte aligned");
  const size_t need = cbk_tree_attn_workspace_bytes(n_nodes, cap, n_q_heads, n_kv_heads, head_dim);
  if (workspace_bytes < need)
    return set_error(CBK_ERR_WORKSPACE, "cbk_tree_attn: workspace %zu < %zu bytes", workspace_bytes, need);
  const dim3 grid(n_nodes, n_q_heads);
  auto st = static_cast<cudaStream_t>(stream);
  const float sl2 = scale * 1.4426950408889634f;
#define CBK_TREE(DT, HD)                                                                                           \
  tree_attn_kernel<DT, HD><<<grid, kTreeThreads, 0, st>>>(                                                         \
      static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k_cache), static_cast<const uint16_t*>(v_cache), \
      kv_row_stride, n_ctx, reinterpret_cast<const uint32_t*>(words), words_stride, n_nodes, cap, n_q_heads,       \
      n_q_heads / n_kv_heads, sl2, static_cast<uint16_t*>(out), status)
  if (dtype == CBK_BF16) {
    if (head_dim == 128) CBK_TREE(CBK_BF16, 128); else CBK_TREE(CBK_BF16, 64);
  } else {
    if (head_dim == 128) CBK_TREE(CBK_F16, 128); else CBK_TREE(CBK_F16, 64);
  }
#undef CBK_TREE
  return check_launch("tree_attn_kernel");
}

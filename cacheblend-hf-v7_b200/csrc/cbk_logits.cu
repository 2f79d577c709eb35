// Penalties for repeated tokens, bias and grammar mask on rows of logits, and the
// token each row chooses, in one pass.
//
// Row r has a history of tokens: its prompt's, then the ones it made (and, when
// the rows are the nodes of a drafted tree, the tokens on the node's own path).
// With c = how often token t was made and "seen" = made or in the prompt:
//   x = logit;  seen:  x = x > 0 ? x / repetition : x * repetition
//   c > 0:      x = x - frequency * c;  x = x - presence
//   x = x + bias[t];  not allowed by the mask:  x = -inf
// in fp32, each step rounded on its own (no contraction), so that rows choose
// what a step-by-step fp32 computation of the same formulas chooses.  The token
// is the first largest x, NaN counting as larger than any number; a row whose
// mask allows nothing is all -inf and chooses token 0.
//
// A cluster of CTAs takes a row, each CTA a contiguous segment of the vocabulary,
// whose counts it keeps in its shared memory (bits 0-30 made, bit 31 in the
// prompt).  The history is read once per row: the CTAs share its positions and
// add to the owner's counts through distributed shared memory.  The row's choice
// is a maximum over 64-bit keys (order of x, then lowest index) in the CTA and
// over the cluster: one launch, no workspace, no order of atomics that could show.
#include <algorithm>

#include "cbk_common.cuh"

namespace cbk {

int ensure_smem_attr(const void* func, int bytes);   // cbk_api.cu

constexpr int kLgThreads = 512;
constexpr int kLgCluster = 8;
constexpr int kLgMaxVocab = kLgCluster * 56 * 1024;   // a segment's counts fit in shared memory
constexpr uint32_t kLgPrompt = 0x80000000u;

struct LogitsParams {
  const void* logits;
  void* out;
  const int64_t *history, *lengths, *n_prompt, *tree_tokens;
  const uint32_t *mask, *tree_words;
  const float* bias;
  int64_t* tokens;
  int32_t* status;
  int64_t row_stride, out_stride, hist_stride, hist_cap, len_stride, prompt_stride, bias_stride, mask_stride,
      tree_stride;
  int rows, vocab, seg, n_tree, counted;
  float repetition, presence, frequency;
};

// order of fp32 values as unsigned integers: -inf < ... < -0 = +0 < ... < inf < NaN
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_rank(uint32_t saddr, uint32_t rank) {
  uint32_t d;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(saddr), "r"(rank));
  return d;
}

template <int DT>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if constexpr (DT == CBK_F32) return static_cast<const float*>(p)[i];
  else return Elem<DT>::to_f(static_cast<const uint16_t*>(p)[i]);
}
template <int DT>
__device__ __forceinline__ void store1(void* p, int64_t i, float x) {
  if constexpr (DT == CBK_F32) static_cast<float*>(p)[i] = x;
  else static_cast<uint16_t*>(p)[i] = Elem<DT>::from_f(x);
}

template <int IN, int OUT>
__global__ void __launch_bounds__(kLgThreads)
process_logits_kernel(const LogitsParams p) {
  extern __shared__ uint32_t s_count[];             // [seg] when the row has a history
  __shared__ unsigned long long s_best[kLgThreads / 32];
  __shared__ unsigned long long s_row[kLgCluster];  // rank 0: one key per CTA of the cluster
  const int row = blockIdx.x / kLgCluster, rank = static_cast<int>(cluster_rank());
  const int tid = threadIdx.x;
  const int v0 = rank * p.seg, v1 = min(v0 + p.seg, p.vocab);

  if (p.counted) {
    for (int i = tid; i < p.seg; i += kLgThreads) s_count[i] = 0;
    cluster_sync_all();                              // every CTA's counts are zero before any is added to
    const uint32_t base = smem_u32(s_count);
    auto add = [&](int64_t t, bool made) {
      if (t < 0 || t >= p.vocab) {
        report(p.status, CBK_STATUS_BAD_INDEX);
        return;
      }
      const int owner = static_cast<int>(t) / p.seg;
      const uint32_t a = map_rank(base + 4u * (static_cast<int>(t) - owner * p.seg), owner);
      if (made) asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(a), "r"(1u) : "memory");
      else asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(a), "r"(kLgPrompt) : "memory");
    };
    if (p.history) {
      int64_t len = p.lengths ? p.lengths[row * p.len_stride] : p.hist_cap;
      if (len < 0 || len > p.hist_cap) {
        if (tid == 0) report(p.status, CBK_STATUS_BAD_INDEX);
        len = len < 0 ? 0 : p.hist_cap;
      }
      const int64_t prompt = p.n_prompt ? p.n_prompt[row * p.prompt_stride] : 0;
      const int64_t* h = p.history + row * p.hist_stride;
      for (int64_t i = rank * kLgThreads + tid; i < len; i += kLgCluster * kLgThreads) add(h[i], i >= prompt);
    }
    for (int j = rank * kLgThreads + tid; j < p.n_tree; j += kLgCluster * kLgThreads)
      if ((p.tree_words[row * p.tree_stride + j / 32] >> (j % 32)) & 1u) add(p.tree_tokens[j], true);
  }
  // counts are whole; and every CTA of the cluster runs before one stores into rank 0
  cluster_sync_all();

  unsigned long long best = 0;
  for (int i = v0 + tid; i < v1; i += kLgThreads) {
    float x = load1<IN>(p.logits, row * p.row_stride + i);
    if (p.counted) {
      const uint32_t n = s_count[i - v0], c = n & ~kLgPrompt;
      if (n) x = x > 0.f ? __fdiv_rn(x, p.repetition) : __fmul_rn(x, p.repetition);
      if (c) x = __fsub_rn(__fsub_rn(x, __fmul_rn(p.frequency, static_cast<float>(c))), p.presence);
    }
    if (p.bias) x = __fadd_rn(x, p.bias[row * p.bias_stride + i]);
    if (p.mask && !((p.mask[row * p.mask_stride + i / 32] >> (i % 32)) & 1u)) x = -INFINITY;
    if (p.out) store1<OUT>(p.out, row * p.out_stride + i, x);
    const unsigned long long k = (static_cast<unsigned long long>(order_key(x)) << 32) | (0xffffffffu - i);
    best = k > best ? k : best;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long k = __shfl_xor_sync(0xffffffffu, best, o);
    best = k > best ? k : best;
  }
  if ((tid & 31) == 0) s_best[tid >> 5] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kLgThreads / 32; ++w) best = s_best[w] > best ? s_best[w] : best;
    const uint32_t a = map_rank(smem_u32(&s_row[rank]), 0);
    asm volatile("st.relaxed.cluster.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(best) : "memory");
  }
  cluster_sync_all();
  if (rank == 0 && tid == 0) {
    best = s_row[0];
    for (int c = 1; c < kLgCluster; ++c) best = s_row[c] > best ? s_row[c] : best;
    p.tokens[row] = 0xffffffffu - static_cast<uint32_t>(best);
  }
}

template <int IN, int OUT>
static int launch_logits(const LogitsParams& p, cudaStream_t st) {
  auto kern = process_logits_kernel<IN, OUT>;
  const int smem = p.counted ? p.seg * 4 : 0;
  if (smem > 48 * 1024)
    if (int rc = ensure_smem_attr(reinterpret_cast<const void*>(kern), 224 * 1024)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows) * kLgCluster);
  cfg.blockDim = dim3(kLgThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kLgCluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) return set_error(CBK_ERR_CUDA, "process_logits_kernel launch: %s", cudaGetErrorString(e));
  return check_launch("process_logits_kernel");
}

}  // namespace cbk

using namespace cbk;

extern "C" int cbk_process_logits(const cbk_process_logits_args* a, void* stream) {
  if (!a || a->size != sizeof(*a)) return set_error(CBK_ERR_INVALID, "cbk_process_logits: bad argument struct");
  if (a->in_dtype != CBK_BF16 && a->in_dtype != CBK_F16 && a->in_dtype != CBK_F32)
    return set_error(CBK_ERR_UNSUPPORTED, "cbk_process_logits: dtype %d not supported", a->in_dtype);
  if (a->out && a->out_dtype != a->in_dtype && a->out_dtype != CBK_F32)
    return set_error(CBK_ERR_UNSUPPORTED, "cbk_process_logits: output dtype %d for input dtype %d (the same or fp32)",
                     a->out_dtype, a->in_dtype);
  if (a->vocab <= 0 || a->vocab > kLgMaxVocab)
    return set_error(CBK_ERR_UNSUPPORTED, "cbk_process_logits: vocabulary %lld (1 to %d)", (long long)a->vocab,
                     kLgMaxVocab);
  if (a->rows < 0 || a->rows > (1 << 24))
    return set_error(CBK_ERR_INVALID, "cbk_process_logits: %lld rows", (long long)a->rows);
  if (a->rows == 0) return CBK_OK;
  if (!a->logits || !a->tokens) return set_error(CBK_ERR_INVALID, "cbk_process_logits: null pointer argument");
  if (!(a->repetition > 0.f)) return set_error(CBK_ERR_INVALID, "cbk_process_logits: repetition penalty must be > 0");
  if (a->presence != a->presence || a->frequency != a->frequency)
    return set_error(CBK_ERR_INVALID, "cbk_process_logits: presence / frequency penalty is NaN");
  if (a->row_stride < a->vocab || (a->out && a->out_stride < a->vocab) ||
      (a->mask && a->mask_stride != 0 && a->mask_stride < (a->vocab + 31) / 32) ||
      (a->bias && a->bias_stride != 0 && a->bias_stride < a->vocab))
    return set_error(CBK_ERR_INVALID, "cbk_process_logits: row stride shorter than a row");
  if (a->history_cap < 0 || a->history_cap >= (int64_t{1} << 30) || a->n_tree < 0 || a->n_tree > 1024 ||
      (a->n_tree > 0 && (!a->tree_tokens || !a->tree_words || a->tree_stride < (a->n_tree + 31) / 32)))
    return set_error(CBK_ERR_INVALID, "cbk_process_logits: bad history or tree");
  LogitsParams p;
  p.logits = a->logits;
  p.out = a->out;
  p.history = a->history_cap > 0 ? a->history : nullptr;
  p.lengths = a->lengths;
  p.n_prompt = a->n_prompt;
  p.tree_tokens = a->tree_tokens;
  p.mask = reinterpret_cast<const uint32_t*>(a->mask);
  p.tree_words = reinterpret_cast<const uint32_t*>(a->tree_words);
  p.bias = a->bias;
  p.tokens = a->tokens;
  p.status = a->status;
  p.row_stride = a->row_stride;
  p.out_stride = a->out_stride;
  p.hist_stride = a->history_stride;
  p.hist_cap = a->history_cap;
  p.len_stride = a->lengths_stride;
  p.prompt_stride = a->n_prompt_stride;
  p.bias_stride = a->bias_stride;
  p.mask_stride = a->mask_stride;
  p.tree_stride = a->tree_stride;
  p.rows = static_cast<int>(a->rows);
  p.vocab = static_cast<int>(a->vocab);
  p.seg = static_cast<int>((a->vocab + kLgCluster * 32 - 1) / (kLgCluster * 32) * 32);
  p.n_tree = a->n_tree;
  p.counted = p.history != nullptr || a->n_tree > 0;
  p.repetition = a->repetition;
  p.presence = a->presence;
  p.frequency = a->frequency;
  auto st = static_cast<cudaStream_t>(stream);
  const bool f32 = a->out && a->out_dtype == CBK_F32;
  switch (a->in_dtype) {
    case CBK_F32: return launch_logits<CBK_F32, CBK_F32>(p, st);
    case CBK_BF16: return f32 ? launch_logits<CBK_BF16, CBK_F32>(p, st) : launch_logits<CBK_BF16, CBK_BF16>(p, st);
    default: return f32 ? launch_logits<CBK_F16, CBK_F32>(p, st) : launch_logits<CBK_F16, CBK_F16>(p, st);
  }
}

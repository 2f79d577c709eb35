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
// A cluster of CTAs takes a row (several rows, one after the other, when there are
// more rows than clusters fit), each CTA a contiguous segment of the vocabulary,
// whose counts it keeps in its shared memory (bits 0-30 made, bit 31 in the
// prompt).  The history is read once per row -- once per cluster when the rows
// share it -- the CTAs sharing its positions and adding to the owner's counts
// through distributed shared memory; a tree node's path is added for its row and
// taken back after it.  The row's choice is a maximum over 64-bit keys (order of x,
// then lowest index) in the CTA and over the cluster: one launch, no workspace, no
// order of atomics that could show.
//
// Bound by memory for many rows, by latency for few: a thread takes vectors of 8
// logits (16 or 32 bytes), kLgBatch loads in flight, the first batch before the
// counting starts.  Rows that do not lie on 16-byte boundaries are read element by
// element, neighbouring lanes on neighbouring elements.
#include <algorithm>

#include "cbk_common.cuh"

namespace cbk {

int ensure_smem_attr(const void* func, int bytes);   // cbk_api.cu

constexpr int kLgThreads = 512;
constexpr int kLgCluster = 8;
constexpr int kLgBatch = 4;
constexpr int kLgBlock = 128;                           // tokens of a CTA's blocks
constexpr int kLgMaxClusters = 36;                      // two CTAs on each of 148 SMs, whole clusters
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
  int rows, vocab, seg, n_tree, counted, shared;
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

// max that propagates NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// VEC consecutive logits of a row as they lie in memory
template <int DT, int VEC>
struct Raw {
  static constexpr int kWords = DT == CBK_F32 ? VEC : (VEC + 1) / 2;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    if constexpr (VEC == 8) {
      const uint4* v = reinterpret_cast<const uint4*>(static_cast<const char*>(p) + i * (DT == CBK_F32 ? 4 : 2));
#pragma unroll
      for (int k = 0; k < kWords / 4; ++k) {
        const uint4 x = v[k];
        w[4 * k] = x.x;
        w[4 * k + 1] = x.y;
        w[4 * k + 2] = x.z;
        w[4 * k + 3] = x.w;
      }
    } else if constexpr (DT == CBK_F32) {
      w[0] = static_cast<const uint32_t*>(p)[i];
    } else {
      w[0] = static_cast<const uint16_t*>(p)[i];
    }
  }
  __device__ __forceinline__ float at(int e) const {
    if constexpr (DT == CBK_F32) return __uint_as_float(w[e]);
    else return Elem<DT>::to_f(static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1))));
  }
};

template <int IN, int OUT, int VEC>
__global__ void __launch_bounds__(kLgThreads, 2)
process_logits_kernel(const LogitsParams p) {
  constexpr int kBatch = VEC == 1 ? 8 : IN == CBK_F32 ? kLgBatch / 2 : kLgBatch;
  extern __shared__ __align__(16) uint32_t s_count[];    // [seg] when the rows have a history
  __shared__ unsigned long long s_best[kLgThreads / 32];
  __shared__ unsigned long long s_row[kLgCluster];       // rank 0: one key per CTA of the cluster
  const int rank = static_cast<int>(cluster_rank()), tid = threadIdx.x;
  const int n_clusters = gridDim.x / kLgCluster;
  // the CTA's share of the vocabulary: every kLgCluster-th block of kLgBlock tokens,
  // one after the other at offsets [0, seg) of its counts
  auto token_at = [&](int o) { return ((o / kLgBlock) * kLgCluster + rank) * kLgBlock + o % kLgBlock; };
  auto add = [&](int64_t t, bool made, uint32_t by) {
    if (t < 0 || t >= p.vocab) {
      if (rank == 0) report(p.status, CBK_STATUS_BAD_INDEX);
      return;
    }
    const uint32_t block = static_cast<uint32_t>(t) / kLgBlock;
    const uint32_t o = (block / kLgCluster) * kLgBlock + static_cast<uint32_t>(t) % kLgBlock;
    if (block % kLgCluster != rank) return;
    if (made) atomicAdd(s_count + o, by);
    else atomicOr(s_count + o, kLgPrompt);
  };
  auto add_path = [&](int row, uint32_t by) {
    for (int j = tid; j < p.n_tree; j += kLgThreads)
      if ((p.tree_words[row * p.tree_stride + j / 32] >> (j % 32)) & 1u) add(p.tree_tokens[j], true, by);
  };

  for (int row = blockIdx.x / kLgCluster, turn = 0; row < p.rows; row += n_clusters, ++turn) {
    const char* in_row = static_cast<const char*>(p.logits) + row * p.row_stride * (IN == CBK_F32 ? 4 : 2);
    // offset of the thread's vector k of batch b: neighbouring lanes on neighbouring vectors
    auto offset = [&](int b, int k) { return ((b * kBatch + k) * kLgThreads + tid) * VEC; };
    Raw<IN, VEC> raw[kBatch];
    auto load_batch = [&](int b) {
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int o = offset(b, k), i = token_at(o);
        if (o < p.seg && i + VEC <= p.vocab) raw[k].load(in_row, i);
      }
    };
    load_batch(0);

    if (p.counted) {
      if (turn == 0 || !p.shared) {
        for (int i = tid; i < p.seg / 4; i += kLgThreads) reinterpret_cast<uint4*>(s_count)[i] = make_uint4(0, 0, 0, 0);
        cluster_sync_all();                          // every CTA's counts are zero before any is added to
        if (p.history) {
          int64_t len = p.lengths ? p.lengths[row * p.len_stride] : p.hist_cap;
          const int64_t prompt = p.n_prompt ? p.n_prompt[row * p.prompt_stride] : 0;
          if (len < 0 || len > p.hist_cap) {
            if (tid == 0) report(p.status, CBK_STATUS_BAD_INDEX);
            len = len < 0 ? 0 : p.hist_cap;
          }
          const int64_t* h = p.history + row * p.hist_stride;
          constexpr int kAhead = 8;
          for (int64_t i = tid; i < len; i += kAhead * kLgThreads) {
            int64_t t[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) t[k] = i + k * kLgThreads < len ? __ldg(h + i + k * kLgThreads) : 0;
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
              if (i + k * kLgThreads < len) add(t[k], i + k * kLgThreads >= prompt, 1u);
          }
        }
        add_path(row, 1u);
      } else {
        // the last row's reads of the counts lie behind its closing cluster barrier
        add_path(row - n_clusters, 0xffffffffu);
        add_path(row, 1u);
      }
    }
    // counts are whole; and every CTA of the cluster runs before one stores into rank 0
    cluster_sync_all();

    float best = -INFINITY;
    int best_i = token_at(tid * VEC);                     // the thread's first element: the first of a row of -inf
    auto finish = [&](float x, int i) {              // everything but the penalties, then the store
      if (p.mask && !((p.mask[row * p.mask_stride + i / 32] >> (i % 32)) & 1u)) x = -INFINITY;
      return x;
    };
    auto penalise = [&](float x, uint32_t n) {
      if (n) {
        x = x > 0.f ? __fdiv_rn(x, p.repetition) : __fmul_rn(x, p.repetition);
        const uint32_t c = n & ~kLgPrompt;
        if (c) x = __fsub_rn(__fsub_rn(x, __fmul_rn(p.frequency, static_cast<float>(c))), p.presence);
      }
      return x;
    };
    auto take = [&](float x, int i) {
      if (x > best || (x != x && best == best)) {
        best = x;
        best_i = i;
      }
    };
    const int n_batches = (p.seg + kBatch * kLgThreads * VEC - 1) / (kBatch * kLgThreads * VEC);
    for (int b = 0; b < n_batches; ++b) {
      if (b > 0) load_batch(b);
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int o = offset(b, k), i = token_at(o);
        if (o >= p.seg || i >= p.vocab) continue;
        if (VEC == 8 && i + VEC <= p.vocab) {
          float x[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) x[e] = raw[k].at(e);
          if (p.counted) {
            uint32_t n[VEC], any = 0;
#pragma unroll
            for (int q = 0; q < VEC / 4; ++q) {
              const uint4 c4 = *reinterpret_cast<const uint4*>(s_count + o + 4 * q);
              n[4 * q] = c4.x;
              n[4 * q + 1] = c4.y;
              n[4 * q + 2] = c4.z;
              n[4 * q + 3] = c4.w;
              any |= c4.x | c4.y | c4.z | c4.w;
            }
            if (any) {
#pragma unroll
              for (int e = 0; e < VEC; ++e) x[e] = penalise(x[e], n[e]);
            }
          }
          if (p.bias) {
            const float4* bv = reinterpret_cast<const float4*>(p.bias + row * p.bias_stride + i);
#pragma unroll
            for (int q = 0; q < VEC / 4; ++q) {
              const float4 c4 = __ldg(bv + q);
              x[4 * q] = __fadd_rn(x[4 * q], c4.x);
              x[4 * q + 1] = __fadd_rn(x[4 * q + 1], c4.y);
              x[4 * q + 2] = __fadd_rn(x[4 * q + 2], c4.z);
              x[4 * q + 3] = __fadd_rn(x[4 * q + 3], c4.w);
            }
          }
          if (p.mask) {
            // i is a multiple of 8: the 8 bits are one byte of the row
            const uint32_t bits = __ldg(reinterpret_cast<const uint8_t*>(p.mask + row * p.mask_stride) + i / 8);
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[e] = (bits >> e) & 1u ? x[e] : -INFINITY;
          }
          float m = x[0];
#pragma unroll
          for (int e = 1; e < VEC; ++e) m = max_nan(m, x[e]);
          if (!(m <= best)) {                        // larger, or NaN: rare after the first few
#pragma unroll
            for (int e = 0; e < VEC; ++e) take(x[e], i + e);
          }
          if (p.out) {
            if constexpr (OUT == CBK_F32) {
              float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.out) + row * p.out_stride + i);
              dst[0] = make_float4(x[0], x[1], x[2], x[3]);
              dst[1] = make_float4(x[4], x[5], x[6], x[7]);
            } else {
              st_vec(static_cast<uint16_t*>(p.out) + row * p.out_stride + i,
                     make_uint4(Pk<OUT>::cvt(x[0], x[1]), Pk<OUT>::cvt(x[2], x[3]), Pk<OUT>::cvt(x[4], x[5]),
                                Pk<OUT>::cvt(x[6], x[7])));
            }
          }
        } else {
          // a row's last, partial vector, or a row off the boundaries
          for (int j = i; j < min(i + VEC, p.vocab); ++j) {
            float x = VEC == 1 ? raw[k].at(0) : load1<IN>(in_row, j);
            if (p.counted) x = penalise(x, s_count[o + j - i]);
            if (p.bias) x = __fadd_rn(x, p.bias[row * p.bias_stride + j]);
            x = finish(x, j);
            take(x, j);
            if (p.out) store1<OUT>(p.out, row * p.out_stride + j, x);
          }
        }
      }
    }
    // a thread without an element has index >= vocab or another's: it must not win
    unsigned long long key = tid * VEC < p.seg && best_i < p.vocab
        ? (static_cast<unsigned long long>(order_key(best)) << 32) | (0xffffffffu - static_cast<uint32_t>(best_i)) : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
      key = other > key ? other : key;
    }
    if ((tid & 31) == 0) s_best[tid >> 5] = key;
    __syncthreads();
    if (tid < 32) {
      key = tid < kLgThreads / 32 ? s_best[tid] : 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
        key = other > key ? other : key;
      }
      if (tid == 0) {
        const uint32_t a = map_rank(smem_u32(&s_row[rank]), 0);
        asm volatile("st.relaxed.cluster.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(key) : "memory");
      }
    }
    cluster_sync_all();
    if (rank == 0 && tid == 0) {
      key = s_row[0];
      for (int c = 1; c < kLgCluster; ++c) key = s_row[c] > key ? s_row[c] : key;
      p.tokens[row] = 0xffffffffu - static_cast<uint32_t>(key);
    }
  }
}

template <int IN, int OUT, int VEC>
static int launch_logits(const LogitsParams& p, cudaStream_t st) {
  auto kern = process_logits_kernel<IN, OUT, VEC>;
  const int smem = p.counted ? p.seg * 4 : 0;
  if (smem > 48 * 1024)
    if (int rc = ensure_smem_attr(reinterpret_cast<const void*>(kern), 224 * 1024)) return rc;
  cudaLaunchConfig_t cfg = {};
  const int turns = (p.rows + kLgMaxClusters - 1) / kLgMaxClusters;      // rows per cluster
  cfg.gridDim = dim3(static_cast<unsigned>((p.rows + turns - 1) / turns) * kLgCluster);
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
  p.seg = static_cast<int>((a->vocab + kLgCluster * kLgBlock - 1) / (kLgCluster * kLgBlock) * kLgBlock);
  p.n_tree = a->n_tree;
  p.counted = p.history != nullptr || a->n_tree > 0;
  p.shared = p.history == nullptr || (a->history_stride == 0 && a->lengths_stride == 0 && a->n_prompt_stride == 0);
  p.repetition = a->repetition;
  p.presence = a->presence;
  p.frequency = a->frequency;
  auto st = static_cast<cudaStream_t>(stream);
  const bool f32 = a->out && a->out_dtype == CBK_F32;
  // whole 16-byte vectors: every row of logits, output and bias starts on a boundary
  const int in_size = a->in_dtype == CBK_F32 ? 4 : 2, out_size = f32 ? 4 : in_size;
  const uint64_t off = reinterpret_cast<uintptr_t>(a->logits) | (a->rows > 1 ? a->row_stride * in_size : 0) |
                       (a->out ? reinterpret_cast<uintptr_t>(a->out) | (a->rows > 1 ? a->out_stride * out_size : 0) : 0) |
                       (a->bias ? reinterpret_cast<uintptr_t>(a->bias) | (a->bias_stride * 4) : 0);
  const bool vec = (off & 15u) == 0;
#define CBK_LG(IN, OUT) return vec ? launch_logits<IN, OUT, 8>(p, st) : launch_logits<IN, OUT, 1>(p, st)
  switch (a->in_dtype) {
    case CBK_F32: CBK_LG(CBK_F32, CBK_F32);
    case CBK_BF16:
      if (f32) CBK_LG(CBK_BF16, CBK_F32);
      CBK_LG(CBK_BF16, CBK_BF16);
    default:
      if (f32) CBK_LG(CBK_F16, CBK_F32);
      CBK_LG(CBK_F16, CBK_F16);
  }
#undef CBK_LG
}

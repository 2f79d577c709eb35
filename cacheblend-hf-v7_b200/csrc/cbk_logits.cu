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
// process_logits_kernel: a cluster of CTAs takes a row (several rows, one after the
// other, when there are more rows than clusters fit), each CTA every n-th block of
// 128 tokens of the vocabulary.  A thread takes one vector of 8 logits (16 or 32 bytes)
// at a time, with its counts and mask bits loaded beside it, the first one before any
// counting; 32 warps to an SM hide the latency better than more vectors a thread did (2
// and 4 vectors: the same and 10 % slower).  The row's choice is a maximum over 64-bit
// keys (order of x, then lowest index) in the CTA and over the cluster, so no order of
// atomics shows.  Rows that do not lie on 16-byte boundaries are read element by
// element, neighbouring lanes on neighbouring elements.  64 rows of 128256 after 24 K
// tokens with tree, mask and bias: 26 us, bound by instructions and latency (its bytes
// would take 5.3); 16 rows after 5 K with tree and mask 14, one row of 32000 after 6 K 6.
// Penalties alone, 64 rows of 128256 after 24 K tokens: 23.3 us, 22.7 when no logits are
// written; 64 rows with a history of 5 K each 39.1 (every cluster counts), of 32000 22.1.
//
// Penalties come element by element, each behind a branch, or, with a history long for
// its vocabulary (DENSE), for a whole vector in packed pairs without branches.
//
// Counts per token (bits 0-30 made, bit 31 in the prompt) come about in one of two
// ways.  Few rows, or a history per row: a CTA reads the whole history and counts what
// falls into its share, in its shared memory, with no second launch.  Many rows of one
// history: every cluster would do that again, so count_tokens_kernel does it once, in
// the workspace, and the rows read the counts from L2.  What a drafted tree's node
// adds is a short list per row; a bit per vector of 8 tokens says where to look it up.
#include <algorithm>

#include "cbk_attn_common.cuh"

namespace cbk {

int ensure_smem_attr(const void* func, int bytes);   // cbk_api.cu

constexpr int kLgThreads = 512;
constexpr int kLgBlock = 128;                           // tokens of a CTA's blocks
constexpr int kLgMaxVocab = 458752;
constexpr int kLgMaxTree = 1024;
constexpr int kLgMaxSmem = 224 * 1024;
constexpr int kLgCountCtas = 8;                         // CTAs that count a shared history
// Rows from which a shared history is counted once, and clusters of 8 and of 4 that fit
// side by side, two CTAs to each of 148 SMs (another number of SMs changes the time alone).
// Counted by every cluster against once, us, penalties alone: 128256 tokens after 30000
// 16 rows 23.8 / 16.4, 28 rows 24.2 / 16.8, 64 rows 43.4 / 24.1; after 5000 16 rows 13.3 /
// 13.7, 28 rows 13.8 / 14.6, 32 rows 22.4 / 18.2; after 600 16 rows 10.3 / 11.9, 28 rows
// 10.8 / 12.7, 32 rows 17.6 / 14.8; 32000 tokens after 500 28 rows 6.7 / 7.9, 32 rows
// 10.1 / 8.6.  Beyond kLgFit8 rows once always wins; up to it the history's length
// decides, which lies on the device, and 24 takes some of either.
constexpr int kLgManyRows = 24, kLgFit8 = 30, kLgFit4 = 66;
// A history's room over the vocabulary from which a vector's penalties are computed in
// pairs, seen or not, instead of each behind a branch (penalties alone, 64 rows of 128256: a
// history of 24 K tokens 25.3 us with branches, 23.2 without, 12 K 23.3 and 22.7, 6 K 21.1
// and 22.4, 3 K 19.5 and 21.9; one row of 32000 after 6 K 6.6 and 6.0).  The room alone is
// known to the host: a short history in much room pays the difference.
constexpr int kLgDense = 16;
constexpr uint32_t kLgPrompt = 0x80000000u;

struct LogitsParams {
  const void* logits;
  void* out;
  const int64_t *history, *lengths, *n_prompt, *tree_tokens;
  const uint32_t *mask, *tree_words;
  const float* bias;
  uint32_t* counts;               // a shared history's counts in the workspace, or null
  int64_t* tokens;
  int32_t* status;
  int64_t row_stride, out_stride, hist_stride, hist_cap, len_stride, prompt_stride, bias_stride, mask_stride,
      tree_stride;
  int rows, vocab, seg, n_tree, shared, log_cluster;
  float repetition, inv_repetition, inv_rest, presence, frequency;   // inv_rest: what 1 / repetition has beyond 24 bits
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
  // (not .aligned: lanes of a warp may come here apart)
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
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

// x / b for x > 0, correctly rounded, from y = the rounded 1 / b: q = RN(x y) is
// within two units of the quotient, one correction by its exact remainder brings it
// within one, and then RN(q + (x - q b) y) is the rounded quotient (Markstein,
// "Computation of elementary functions on the IBM RISC System/6000 processor", 1990)
// as long as nothing under- or overflows on the way: y = 0 where b is not between
// 2^-40 and 2^40, and then, or for x outside the range below, the division itself.
__device__ __forceinline__ float divide(float x, float b, float y) {
  if (!(x > 1e-20f && x < 1e20f) || y == 0.f) return __fdiv_rn(x, b);
  float q = __fmul_rn(x, y);
  q = __fmaf_rn(__fmaf_rn(-q, b, x), y, q);
  return __fmaf_rn(__fmaf_rn(-q, b, x), y, q);
}

// one seen element's penalties
__device__ __forceinline__ float penalise1(float x, uint32_t n, float rep, float inv, float freq, float pres) {
  x = x > 0.f ? divide(x, rep, inv) : __fmul_rn(x, rep);
  const uint32_t c = n & ~kLgPrompt;
  return c ? __fsub_rn(__fsub_rn(x, __fmul_rn(freq, static_cast<float>(c))), pres) : x;
}
// (as a call, where it is the rare case and would only fill the instruction cache)
__device__ __noinline__ float penalise_apart(float x, uint32_t n, float rep, float inv, float freq, float pres) {
  return penalise1(x, n, rep, inv, freq, pres);
}

// whether the magnitudes of 8 numbers are in divide's range
__device__ __forceinline__ bool in_range(const float* x) {
  const float hi = max3f(max3f(fabsf(x[0]), fabsf(x[1]), fabsf(x[2])), max3f(fabsf(x[3]), fabsf(x[4]), fabsf(x[5])),
                         fmaxf(fabsf(x[6]), fabsf(x[7])));
  float lo = fminf(fabsf(x[0]), fabsf(x[1]));
#pragma unroll
  for (int e = 2; e < 8; ++e) lo = fminf(lo, fabsf(x[e]));
  return lo > 1e-20f && hi < 1e20f;
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

// One cluster: clear the counts, then add the tokens of the history that all rows share.
__global__ void __launch_bounds__(1024)
count_tokens_kernel(const LogitsParams p) {
  const int rank = static_cast<int>(cluster_rank());
  const int tid = rank * 1024 + threadIdx.x;
  constexpr int kStep = kLgCountCtas * 1024;
  uint32_t* counts = p.counts;
  const int cells = (p.vocab + 127) / 128 * 128;
  for (int i = tid; i < cells / 4; i += kStep)
    reinterpret_cast<uint4*>(counts)[i] = make_uint4(0, 0, 0, 0);
  int64_t len = p.lengths ? *p.lengths : p.hist_cap;
  const int64_t prompt = p.n_prompt ? *p.n_prompt : 0;
  if (len < 0 || len > p.hist_cap) {
    if (tid == 0) report(p.status, CBK_STATUS_BAD_INDEX);
    len = len < 0 ? 0 : p.hist_cap;
  }
  const int64_t* h = p.history;
  constexpr int kAhead = 4;
  bool cleared = false, bad = false;
  for (int64_t i0 = 0; i0 < len; i0 += kAhead * kStep) {
    int64_t t[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (i0 + k * kStep + tid < len) t[k] = __ldg(h + i0 + k * kStep + tid);
    if (!cleared) cluster_sync_all();                 // every count is zero before any is added to
    cleared = true;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t i = i0 + k * kStep + tid;
      if (i >= len) break;
      if (t[k] < 0 || t[k] >= p.vocab) bad = true;
      else if (i >= prompt) atomicAdd(counts + t[k], 1u);
      else atomicOr(counts + t[k], kLgPrompt);
    }
  }
  if (bad) report(p.status, CBK_STATUS_BAD_INDEX);
  grid_launch_dependents();
}

template <int IN, int OUT, int VEC, bool DENSE>
__global__ void __launch_bounds__(kLgThreads, 2)
process_logits_kernel(const LogitsParams p) {
  constexpr int kBatch = VEC == 1 ? 8 : 1;
  // counts [seg] (when the CTA counts), path bits [seg / 256] and path [n_tree] (with a tree)
  extern __shared__ __align__(16) uint32_t s_dyn[];
  __shared__ int s_n_path;
  __shared__ unsigned long long s_best[kLgThreads / 32];
  __shared__ unsigned long long s_row[16];               // rank 0: one key per CTA of the cluster
  const int rank = static_cast<int>(cluster_rank()), tid = threadIdx.x;
  const int n_clusters = gridDim.x >> p.log_cluster, cluster_mask = (1 << p.log_cluster) - 1;
  const bool counts_here = p.history != nullptr && p.counts == nullptr;
  uint32_t* s_count = s_dyn;
  uint32_t* s_over = s_dyn + (counts_here ? p.seg : 0);
  uint32_t* s_path = s_over + (p.n_tree > 0 ? (p.seg + 255) / 256 : 0);

  // the CTA's share of the vocabulary: every n-th block of kLgBlock tokens, one after
  // the other at offsets [0, seg)
  auto token_at = [&](int o) { return (((o / kLgBlock) << p.log_cluster) + rank) * kLgBlock + o % kLgBlock; };
  auto offset_of = [&](uint32_t t) {
    return static_cast<int>(((t / kLgBlock) >> p.log_cluster) * kLgBlock + t % kLgBlock);
  };
  // (the low word alone says whose token it is; one outside the vocabulary is reported by one CTA)
  auto ours = [&](int64_t t) { return (static_cast<int>(static_cast<uint32_t>(t) / kLgBlock) & cluster_mask) == rank; };
  auto known = [&](int64_t t) {
    if (static_cast<uint64_t>(t) < static_cast<uint64_t>(p.vocab)) return true;
    report(p.status, CBK_STATUS_BAD_INDEX);
    return false;
  };
  auto add = [&](int64_t t, bool made) {
    if (!known(t)) return;
    if (made) atomicAdd(s_count + offset_of(static_cast<uint32_t>(t)), 1u);
    else atomicOr(s_count + offset_of(static_cast<uint32_t>(t)), kLgPrompt);
  };
  if (p.n_tree > 0) {
    for (int i = tid; i < (p.seg + 255) / 256; i += kLgThreads) s_over[i] = 0;
    if (tid == 0) s_n_path = 0;
    __syncthreads();
  }

  for (int row = blockIdx.x >> p.log_cluster, turn = 0; row < p.rows; row += n_clusters, ++turn) {
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

    for (int j = tid; j < p.n_tree; j += kLgThreads)
      if ((p.tree_words[row * p.tree_stride + j / 32] >> (j % 32)) & 1u) {
        const int64_t t = p.tree_tokens[j];
        if (!ours(t) || !known(t)) continue;
        const int o = offset_of(static_cast<uint32_t>(t));
        s_path[atomicAdd(&s_n_path, 1)] = o;
        atomicOr(s_over + o / 256, 1u << (o / 8 % 32));
      }
    if (counts_here && (turn == 0 || !p.shared)) {
      for (int i = tid; i < p.seg / 4; i += kLgThreads) reinterpret_cast<uint4*>(s_count)[i] = make_uint4(0, 0, 0, 0);
      int64_t len = p.lengths ? p.lengths[row * p.len_stride] : p.hist_cap;
      const int64_t prompt = p.n_prompt ? p.n_prompt[row * p.prompt_stride] : 0;
      if (len < 0 || len > p.hist_cap) {
        if (rank == 0 && tid == 0) report(p.status, CBK_STATUS_BAD_INDEX);
        len = len < 0 ? 0 : p.hist_cap;
      }
      const int64_t* h = p.history + row * p.hist_stride;
      __syncthreads();
      constexpr int kAhead = 8;
      for (int64_t i = tid; i < len; i += kAhead * kLgThreads) {
        int64_t t[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) t[k] = i + k * kLgThreads < len ? __ldg(h + i + k * kLgThreads) : 0;
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
          if (i + k * kLgThreads < len && ours(t[k])) add(t[k], i + k * kLgThreads >= prompt);
      }
    }
    if (p.counts && turn == 0) grid_wait();          // a dependent of count_tokens_kernel: its counts are whole
    __syncthreads();
    // every CTA of the cluster runs before one stores into rank 0
    if (turn == 0) cluster_sync_all();

    float best = -INFINITY;
    int best_i = token_at(tid * VEC);                     // the thread's first element: the first of a row of -inf
    auto penalise = [&](float x, uint32_t n) {
      if (!n) return x;
      if constexpr (DENSE) return penalise_apart(x, n, p.repetition, p.inv_repetition, p.frequency, p.presence);
      else return penalise1(x, n, p.repetition, p.inv_repetition, p.frequency, p.presence);
    };
    // the same for a vector, in pairs and without branches.  With y + y_rest = 1 / rep to
    // twice the bits the first q is within one unit of the quotient, and divide's last
    // step makes it the rounded one.
    auto penalise8 = [&](float* x, const uint32_t* n) {
      const uint64_t y = pk_f2(p.inv_repetition, p.inv_repetition), y_rest = pk_f2(p.inv_rest, p.inv_rest);
      const uint64_t rep = pk_f2(p.repetition, p.repetition), neg_rep = pk_f2(-p.repetition, -p.repetition);
      const uint64_t neg_magic = pk_f2(-8388608.f, -8388608.f);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const uint64_t v = pk_f2(x[e], x[e + 1]);
        uint64_t q = fma_f2(v, y, mul_f2(v, y_rest));
        q = fma_f2(fma_f2(q, neg_rep, v), y, q);
        float a[2], b[2];
        upk_f2(q, a[0], a[1]);
        upk_f2(mul_f2(v, rep), b[0], b[1]);
        uint64_t z = pk_f2(x[e] > 0.f ? a[0] : b[0], x[e + 1] > 0.f ? a[1] : b[1]);
        // c < 2^23 as a float: 2^23 + c has c's bits in its mantissa
        const uint32_t c0 = n[e] & ~kLgPrompt, c1 = n[e + 1] & ~kLgPrompt;
        upk_f2(add_f2(pk_f2(__uint_as_float(c0 | 0x4b000000u), __uint_as_float(c1 | 0x4b000000u)), neg_magic), b[0], b[1]);
        // (a packed product would be contracted with the sum, which then rounds once)
        z = add_f2(z, pk_f2(__fmul_rn(-p.frequency, b[0]), __fmul_rn(-p.frequency, b[1])));
        z = add_f2(z, pk_f2(c0 ? -p.presence : 0.f, c1 ? -p.presence : 0.f));
        upk_f2(z, a[0], a[1]);
        x[e] = n[e] ? a[0] : x[e];
        x[e + 1] = n[e + 1] ? a[1] : x[e + 1];
      }
    };
    auto take = [&](float x, int i) {
      if (x > best || (x != x && best == best)) {
        best = x;
        best_i = i;
      }
    };
    const int n_path = p.n_tree > 0 ? s_n_path : 0;
    const bool paired = DENSE && p.inv_repetition != 0.f && fabsf(p.presence) < INFINITY &&
                        fabsf(p.frequency) < INFINITY;
    auto on_path = [&](int o) { return n_path > 0 && ((s_over[o / 256] >> (o / 8 % 32)) & 1u); };
    const int n_batches = (p.seg + kBatch * kLgThreads * VEC - 1) / (kBatch * kLgThreads * VEC);
    for (int b = 0; b < n_batches; ++b) {
      if (b > 0) load_batch(b);
      // the vector's counts and mask bits on their way beside it
      uint4 c_lo = make_uint4(0, 0, 0, 0), c_hi = c_lo;
      uint32_t bits = 0xffu;
      if (VEC == 8) {
        const int o = offset(b, 0), i = token_at(o);
        if (o < p.seg && i + VEC <= p.vocab) {
          if (p.counts) {
            c_lo = *reinterpret_cast<const uint4*>(p.counts + i);
            c_hi = *reinterpret_cast<const uint4*>(p.counts + i + 4);
          }
          // i is a multiple of 8: the 8 bits are one byte of the row
          if (p.mask) bits = __ldg(reinterpret_cast<const uint8_t*>(p.mask + row * p.mask_stride) + i / 8);
        }
      }
      // element by element: a batch of them, with all that belongs to each on its way
      // beside it (5 rows of 32003: 9.0 -> 7.6 us)
      uint32_t n1[kBatch], m1[kBatch];
      float b1[kBatch];
      if (VEC == 1) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int o = offset(b, k), i = token_at(o);
          const bool in = o < p.seg && i < p.vocab;
          n1[k] = in && p.counts ? p.counts[i] : in && counts_here ? s_count[o] : 0u;
          m1[k] = in && p.mask ? p.mask[row * p.mask_stride + i / 32] : 0xffffffffu;
          b1[k] = in && p.bias ? p.bias[row * p.bias_stride + i] : 0.f;
        }
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int o = offset(b, k), i = token_at(o);
        if (o >= p.seg || i >= p.vocab) continue;
        if constexpr (VEC == 1) {
          uint32_t n = n1[k];
          if (on_path(o))
            for (int q = 0; q < n_path; ++q) n += static_cast<int>(s_path[q]) == o ? 1u : 0u;
          float x = penalise(raw[k].at(0), n);
          if (p.bias) x = __fadd_rn(x, b1[k]);
          x = (m1[k] >> (i % 32)) & 1u ? x : -INFINITY;
          take(x, i);
          if (p.out) store1<OUT>(p.out, row * p.out_stride + i, x);
        } else if (i + VEC <= p.vocab) {
          float x[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) x[e] = raw[k].at(e);
          if (p.history || n_path > 0) {
            uint4 lo = c_lo, hi = c_hi;
            if (counts_here) {
              lo = *reinterpret_cast<const uint4*>(s_count + o);
              hi = *reinterpret_cast<const uint4*>(s_count + o + 4);
            }
            uint32_t n[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
            uint32_t any = lo.x | lo.y | lo.z | lo.w | hi.x | hi.y | hi.z | hi.w;
            if (on_path(o)) {
              any = 1;
              for (int j = 0; j < n_path; ++j) {
                const int at = static_cast<int>(s_path[j]) - o;
#pragma unroll
                for (int e = 0; e < VEC; ++e) n[e] += at == e ? 1u : 0u;
              }
              if (DENSE) any = n[0] | n[1] | n[2] | n[3] | n[4] | n[5] | n[6] | n[7];
            }
            if (paired && any && (any & ~kLgPrompt) < (1u << 23) && in_range(x)) {
              penalise8(x, n);
            } else if (any) {
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
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[e] = (bits >> e) & 1u ? x[e] : -INFINITY;
          }
          float m = x[0];
#pragma unroll
          for (int e = 1; e < VEC; ++e) m = max_nan(m, x[e]);
          if (m > best) {                            // the lowest of the equal ones
            int at = VEC - 1;
#pragma unroll
            for (int e = VEC - 2; e >= 0; --e) at = x[e] == m ? e : at;
            best = m;
            best_i = i + at;
          } else if (m != m) {
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
          // a row's last, partial vector
          for (int j = i; j < min(i + VEC, p.vocab); ++j) {
            float x = load1<IN>(in_row, j);
            uint32_t n = p.counts ? p.counts[j] : p.history ? s_count[o + j - i] : 0u;
            if (on_path(o + j - i))
              for (int q = 0; q < n_path; ++q) n += static_cast<int>(s_path[q]) == o + j - i ? 1u : 0u;
            x = penalise(x, n);
            if (p.bias) x = __fadd_rn(x, p.bias[row * p.bias_stride + j]);
            if (p.mask && !((p.mask[row * p.mask_stride + j / 32] >> (j % 32)) & 1u)) x = -INFINITY;
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
    if (p.n_tree > 0) {                              // (the path's readers are behind the barrier above)
      for (int j = tid; j < n_path; j += kLgThreads) s_over[s_path[j] / 256] = 0;
      __syncthreads();
      if (tid == 0) s_n_path = 0;
    }
    cluster_sync_all();
    if (rank == 0 && tid == 0) {
      key = s_row[0];
      for (int c = 1; c <= cluster_mask; ++c) key = s_row[c] > key ? s_row[c] : key;
      p.tokens[row] = 0xffffffffu - static_cast<uint32_t>(key);
    }
    if (row + n_clusters < p.rows) cluster_sync_all();   // read before the next row's choices arrive
  }
}

template <int IN, int OUT, int VEC, bool DENSE>
static int launch_logits(const LogitsParams& p, cudaStream_t st) {
  auto kern = process_logits_kernel<IN, OUT, VEC, DENSE>;
  const int smem = ((p.history && !p.counts ? p.seg : 0) + (p.n_tree > 0 ? (p.seg + 255) / 256 + p.n_tree : 0)) * 4;
  if (int rc = ensure_smem_attr(reinterpret_cast<const void*>(kern), kLgMaxSmem)) return rc;
  if (p.log_cluster > 3) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return set_error(CBK_ERR_CUDA, "process_logits_kernel: %s", cudaGetErrorString(e));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  if (p.counts) {
    attr[0].val.clusterDim.x = kLgCountCtas;
    cfg.gridDim = dim3(kLgCountCtas);
    cfg.blockDim = dim3(1024);
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, count_tokens_kernel, p);
    if (e != cudaSuccess) return set_error(CBK_ERR_CUDA, "count_tokens_kernel launch: %s", cudaGetErrorString(e));
  }
  const int fit = p.log_cluster == 2 ? kLgFit4 : kLgFit8;
  const int turns = (p.rows + fit - 1) / fit, clusters = (p.rows + turns - 1) / turns;
  attr[0].val.clusterDim.x = 1u << p.log_cluster;
  cfg.gridDim = dim3(static_cast<unsigned>(clusters) << p.log_cluster);
  cfg.blockDim = dim3(kLgThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.numAttrs = p.counts ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) return set_error(CBK_ERR_CUDA, "process_logits_kernel launch: %s", cudaGetErrorString(e));
  return check_launch("process_logits_kernel");
}

}  // namespace cbk

using namespace cbk;

// many rows of one history: the counts live in the workspace
static bool counted_once(int64_t rows, int64_t history_stride, int64_t lengths_stride, int64_t n_prompt_stride) {
  return rows >= kLgManyRows && history_stride == 0 && lengths_stride == 0 && n_prompt_stride == 0;
}

extern "C" size_t cbk_process_logits_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows < kLgManyRows || vocab <= 0 || vocab > kLgMaxVocab) return 0;
  return static_cast<size_t>((vocab + 127) / 128 * 128) * sizeof(uint32_t);
}

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
  if (!(a->repetition > 0.f && a->repetition < INFINITY))
    return set_error(CBK_ERR_INVALID, "cbk_process_logits: repetition penalty must be positive and finite");
  if (a->presence != a->presence || a->frequency != a->frequency)
    return set_error(CBK_ERR_INVALID, "cbk_process_logits: presence / frequency penalty is NaN");
  if (a->row_stride < a->vocab || (a->out && a->out_stride < a->vocab) ||
      (a->mask && a->mask_stride != 0 && a->mask_stride < (a->vocab + 31) / 32) ||
      (a->bias && a->bias_stride != 0 && a->bias_stride < a->vocab))
    return set_error(CBK_ERR_INVALID, "cbk_process_logits: row stride shorter than a row");
  if (a->history_cap < 0 || a->history_cap >= (int64_t{1} << 30) || a->n_tree < 0 || a->n_tree > kLgMaxTree ||
      (a->n_tree > 0 && (!a->tree_tokens || !a->tree_words || a->tree_stride < (a->n_tree + 31) / 32)))
    return set_error(CBK_ERR_INVALID, "cbk_process_logits: bad history or tree");
  const bool history = a->history && a->history_cap > 0;
  const bool shared = a->history_stride == 0 && a->lengths_stride == 0 && a->n_prompt_stride == 0;
  const bool once = history && counted_once(a->rows, a->history_stride, a->lengths_stride, a->n_prompt_stride);
  if (once) {
    const size_t need = cbk_process_logits_workspace_bytes(a->rows, a->vocab);
    if (a->workspace_bytes < 0 || static_cast<size_t>(a->workspace_bytes) < need)
      return set_error(CBK_ERR_WORKSPACE, "cbk_process_logits: workspace %lld < %zu bytes",
                       (long long)a->workspace_bytes, need);
    if (!a->workspace || (reinterpret_cast<uintptr_t>(a->workspace) & 15u))
      return set_error(CBK_ERR_INVALID, "cbk_process_logits: the workspace must be 16-byte aligned");
  }
  LogitsParams p;
  p.counts = once ? static_cast<uint32_t*>(a->workspace) : nullptr;
  p.logits = a->logits;
  p.out = a->out;
  p.history = history ? a->history : nullptr;
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
  // clusters of 8 CTAs while all fit side by side, else, with no counts in shared
  // memory, of 4; of 16 where the counts of a large vocabulary would not fit
  p.log_cluster = p.rows > kLgFit8 && (once || !history) ? 2 : 3;
  if (history && !once && (p.vocab / 8 + kLgBlock + p.vocab / 2048 + 2 + kLgMaxTree) * 4 > kLgMaxSmem) p.log_cluster = 4;
  const int span = kLgBlock << p.log_cluster;
  p.seg = (p.vocab + span - 1) / span * kLgBlock;
  p.n_tree = a->n_tree;
  p.shared = shared;
  p.repetition = a->repetition;
  p.inv_repetition = a->repetition >= 0x1p-40f && a->repetition <= 0x1p40f
      ? static_cast<float>(1.0 / static_cast<double>(a->repetition)) : 0.f;
  p.inv_rest = p.inv_repetition == 0.f ? 0.f
      : static_cast<float>(1.0 / static_cast<double>(a->repetition) - static_cast<double>(p.inv_repetition));
  p.presence = a->presence;
  p.frequency = a->frequency;
  auto st = static_cast<cudaStream_t>(stream);
  const bool f32 = a->out && a->out_dtype == CBK_F32;
  // whole 16-byte vectors: every row of logits, output and bias starts on a boundary
  const int in_size = a->in_dtype == CBK_F32 ? 4 : 2, out_size = f32 ? 4 : in_size;
  const uint64_t off = reinterpret_cast<uintptr_t>(a->logits) | (a->rows > 1 ? a->row_stride * in_size : 0) |
                       (a->out ? reinterpret_cast<uintptr_t>(a->out) | (a->rows > 1 ? a->out_stride * out_size : 0) : 0) |
                       (a->bias ? reinterpret_cast<uintptr_t>(a->bias) | (a->bias_stride * 4) : 0);
  const bool vec = (off & 15u) == 0, dense = p.history && a->history_cap * kLgDense >= a->vocab;
#define CBK_LG(IN, OUT)                                                             \
  return !vec ? launch_logits<IN, OUT, 1, false>(p, st)                             \
              : dense ? launch_logits<IN, OUT, 8, true>(p, st) : launch_logits<IN, OUT, 8, false>(p, st)
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

// Per-head RMSNorm and rotation of a step's Q and K, with K and V written into
// their cache rows, in one pass.
//
// For token j (position p = positions[j], cache row r = rows[j]) and a head x of
// D elements: y = x * rsqrt(mean(x^2) + eps) * w (heads of Q and K, when weights
// are given), then the pairs (y_a, y_b) of the first R dimensions -- (i, i + R/2),
// or (2i, 2i + 1) interleaved, i < R/2 -- become (y_a c - y_b s, y_b c + y_a s)
// with (c, s) = table[p][i]; dimensions from R on pass through.  Q goes to
// q_out[j], K to k_cache[r], V unchanged to v_cache[r].
//
// HBM-bound: every byte is read and written once.  A lane owns four pairs of a head
// (8 elements: two 8-byte pieces half a rotation apart, or one 16-byte piece of
// interleaved pairs), so both halves of a pair meet in its registers; LPH = D / 8
// rounded up to a power of two lanes make a head, a warp pass takes 32 / LPH heads
// and kNrUnroll passes are a chunk.  Sources arrive by bulk copies into kNrSlots
// chunks of shared memory per warp, so the bytes in flight cost no registers
// (loads into registers: 171 us for 32768 tokens of 32 + 8 heads of 128, bound by
// the loads' latency at the occupancy the registers left; this way 141 us = 5.8 TB/s,
// 0.89 of measured HBM).  Chunks of 4 passes were 2 % faster there but took 3.8
// instead of 3.1 us for one token; 2, 4 or 8 slots, 4 or 8 CTAs of 256 threads were
// slower, and so was the arithmetic on single floats (158 us: 10 to 20 % more
// instructions, of which a pass of two heads takes 130).  The sum of squares is
// a butterfly within the head's lanes.  A warp takes all heads of a token (several
// warps share one when there are few tokens), so cos, sin and the weights are read
// and multiplied together once per token: with wc = w c, ws = w s and r the root,
//   (z_a, z_b) = ((x_a wc_a - x_b ws_b) r, (x_b wc_b + x_a ws_a) r)
// in packed fp32 pairs.  Everything is fp32 and rounded once at the store
// (CBK_ROPE_FP32), or, in CBK_ROPE_REF, rounded to 16 bits where the HF modules do
// (the normalised value before and after its weight, cos and sin, each product and
// the sum) with packed 16-bit arithmetic.  Without weights that has rope_scatter's bits;
// with them the sum of squares runs in another order than torch's mean, so that a
// normalised value next to a border may round the other way.  32768 tokens of 32 + 8 + 8
// heads of 128 so rounded: 126 us without weights (the decoders' form), 140 with.
#include <algorithm>

#include "cbk_attn_common.cuh"

namespace cbk {

int ensure_smem_attr(const void* func, int bytes);   // cbk_api.cu

constexpr int kNrThreads = 128;
constexpr int kNrWarps = kNrThreads / 32;
constexpr int kNrUnroll = 2;                 // warp passes of a chunk
constexpr int kNrSlots = 3;                  // chunks in flight per warp
constexpr int kNrSlotBytes = kNrUnroll * 512;
constexpr int kNrSmem = kNrWarps * kNrSlots * kNrSlotBytes;
constexpr int64_t kNrFill = 148 * 24;        // warps that fill the GPU: six CTAs of four on each of 148 SMs

struct NormRopeParams {
  const uint16_t *q, *k, *v, *qw, *kw;
  int64_t qs, ks, vs;             // source row strides
  const int64_t *pos, *rows;
  const float4* table;            // (cos, sin) pairs, two per float4
  uint16_t *q_out, *k_cache, *v_cache;
  int32_t* status;
  int64_t n, table_rows, cap, kv_stride;
  int n_q, n_kv, dim, rotary, parts;    // parts: warps per token
  float eps, inv_dim;
};

// a packed 16-bit pair as an fp32 pair
template <int DT>
__device__ __forceinline__ uint64_t widen(uint32_t w) {
  return pk_f2(Elem<DT>::to_f(static_cast<uint16_t>(w)), Elem<DT>::to_f(static_cast<uint16_t>(w >> 16)));
}
template <int DT>
__device__ __forceinline__ uint32_t narrow(uint64_t f2) {
  float lo, hi;
  upk_f2(f2, lo, hi);
  return Pk<DT>::cvt(lo, hi);
}

// a lane's four pairs: a[0], a[1] hold the first elements of pairs (0, 1) and (2, 3), b the second ones
struct Four {
  uint32_t a[2], b[2];
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               :: "r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

template <int DT, int LPH, bool REF, bool PAIRS>
__global__ void __launch_bounds__(kNrThreads, 6)
norm_rope_scatter_kernel(const NormRopeParams p) {
  constexpr int kHeads = 32 / LPH;                   // heads per warp pass
  constexpr int kChunk = kNrUnroll * kHeads;         // heads per chunk
  constexpr unsigned kAll = 0xffffffffu;
  extern __shared__ __align__(128) uint8_t s_rows[];
  __shared__ uint64_t s_bar[kNrWarps][kNrSlots];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t gw = static_cast<int64_t>(blockIdx.x) * kNrWarps + warp;
  const int64_t j = gw / p.parts;
  if (j >= p.n) return;
  const int part = static_cast<int>(gw - j * p.parts);
  // chunks over the heads of Q, then of K, then over V's row in pieces of a slot
  constexpr int kVPiece = kNrSlotBytes / 2;
  const int v_cols = p.n_kv * p.dim;
  const int cq = (p.n_q + kChunk - 1) / kChunk, ck = (p.n_kv + kChunk - 1) / kChunk;
  const int cv = (v_cols + kVPiece - 1) / kVPiece, all = cq + ck + cv;
  const int first = all * part / p.parts, last = all * (part + 1) / p.parts;

  const uint32_t bar0 = smem_u32(&s_bar[warp][0]);
  uint8_t* slots = s_rows + warp * kNrSlots * kNrSlotBytes;
  auto fetch = [&](int c) {                          // chunk c into slot (c - first) % kNrSlots; one lane
    const uint16_t* src;
    int cols;
    if (c < cq) {
      src = p.q + j * p.qs + static_cast<int64_t>(c) * kChunk * p.dim;
      cols = min(kChunk, p.n_q - c * kChunk) * p.dim;
    } else if (c < cq + ck) {
      src = p.k + j * p.ks + static_cast<int64_t>(c - cq) * kChunk * p.dim;
      cols = min(kChunk, p.n_kv - (c - cq) * kChunk) * p.dim;
    } else {
      src = p.v + j * p.vs + static_cast<int64_t>(c - cq - ck) * kVPiece;
      cols = min(kVPiece, v_cols - (c - cq - ck) * kVPiece);
    }
    const int slot = (c - first) % kNrSlots;
    mbar_expect_tx(bar0 + 8 * slot, cols * 2);
    bulk_load(smem_u32(slots + slot * kNrSlotBytes), src, cols * 2, bar0 + 8 * slot);
  };
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kNrSlots; ++i) mbar_init(bar0 + 8 * i, 1);
    fence_barrier_init();
  }
  grid_wait();
  if (lane == 0) {
    for (int c = first; c < min(last, first + kNrSlots); ++c) fetch(c);
  }
  __syncwarp();
  grid_launch_dependents();
  const int64_t pos = p.pos[j], row = p.rows[j];
  bool failed = false;
  auto landed = [&](int c) {
    if (!__all_sync(kAll, mbar_wait(bar0 + 8 * ((c - first) % kNrSlots), ((c - first) / kNrSlots) & 1))) failed = true;
    return !failed;
  };
  const bool bad = row != -1 && (pos < 0 || pos >= p.table_rows || row < 0 || row >= p.cap);
  if (row == -1 || bad) {                            // padding token, or one that is skipped
    if (bad && part == 0 && lane == 0) report(p.status, CBK_STATUS_BAD_INDEX);
    for (int c = first; c < min(last, first + kNrSlots); ++c) landed(c);      // its copies end before the CTA does
    if (failed) report(p.status, CBK_STATUS_TIMEOUT);
    return;
  }

  const int l = lane & (LPH - 1), half = p.rotary / 2;
  const bool live = 8 * l < p.dim, turns = 8 * l < p.rotary;
  // the lane's elements of a head: [ea, ea + 4) and [eb, eb + 4)
  const int ea = PAIRS || !turns ? 8 * l : 4 * l;
  const int eb = PAIRS || !turns ? 8 * l + 4 : half + 4 * l;
  auto load = [&](const uint16_t* head) {
    Four x;
    if (PAIRS) {
      const uint4 r = *reinterpret_cast<const uint4*>(head + ea);
      // interleaved: word i holds pair i
      x.a[0] = __byte_perm(r.x, r.y, 0x5410);
      x.b[0] = __byte_perm(r.x, r.y, 0x7632);
      x.a[1] = __byte_perm(r.z, r.w, 0x5410);
      x.b[1] = __byte_perm(r.z, r.w, 0x7632);
    } else {
      const uint2 ra = *reinterpret_cast<const uint2*>(head + ea), rb = *reinterpret_cast<const uint2*>(head + eb);
      x.a[0] = ra.x;
      x.a[1] = ra.y;
      x.b[0] = rb.x;
      x.b[1] = rb.y;
    }
    return x;
  };
  auto store = [&](uint16_t* head, const Four& x) {
    if (PAIRS) {
      st_vec(head + ea, make_uint4(__byte_perm(x.a[0], x.b[0], 0x5410), __byte_perm(x.a[0], x.b[0], 0x7632),
                                   __byte_perm(x.a[1], x.b[1], 0x5410), __byte_perm(x.a[1], x.b[1], 0x7632)));
    } else {
      *reinterpret_cast<uint2*>(head + ea) = make_uint2(x.a[0], x.a[1]);
      *reinterpret_cast<uint2*>(head + eb) = make_uint2(x.b[0], x.b[1]);
    }
  };

  int c_now = first;                                 // chunks taken so far
  if (first < cq + ck) {
    // cos and sin of the lane's pairs (1, 0 where nothing turns)
    float4 t0 = make_float4(1.f, 0.f, 1.f, 0.f), t1 = t0;
    if (turns) {
      const float4* t = p.table + (pos * half + 4 * l) / 2;
      t0 = __ldg(t);
      t1 = __ldg(t + 1);
    }
    const bool norm = p.qw != nullptr, full = p.rotary == p.dim;
    const uint64_t c[2] = {pk_f2(t0.x, t0.z), pk_f2(t1.x, t1.z)}, s[2] = {pk_f2(t0.y, t0.w), pk_f2(t1.y, t1.w)};
    const uint32_t c16[2] = {narrow<DT>(c[0]), narrow<DT>(c[1])}, s16[2] = {narrow<DT>(s[0]), narrow<DT>(s[1])};

#pragma unroll 1
    for (int kv = 0; kv < 2; ++kv) {                 // the chunks of Q's row, then of K's
      const int end = min(last, kv ? cq + ck : cq);
      if (c_now >= end) continue;
      uint16_t* dst = kv ? p.k_cache + row * p.kv_stride : p.q_out + j * p.n_q * p.dim;
      const uint16_t* weight = kv ? p.kw : p.qw;
      const int n_heads = kv ? p.n_kv : p.n_q;
      Four w = {{0, 0}, {0, 0}};
      if (norm && live) w = load(weight);
      uint64_t ca[2], cb[2], sa[2], sb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint64_t wa = norm ? widen<DT>(w.a[i]) : pk_f2(1.f, 1.f), wb = norm ? widen<DT>(w.b[i]) : pk_f2(1.f, 1.f);
        ca[i] = mul_f2(wa, c[i]);
        cb[i] = mul_f2(wb, c[i]);
        sa[i] = mul_f2(wa, s[i]);
        sb[i] = mul_f2(wb, s[i]) ^ 0x8000000080000000ull;      // z_a takes - x_b w_b s
      }
      for (; c_now < end; ++c_now) {
        if (!landed(c_now)) break;
        const uint16_t* chunk = reinterpret_cast<const uint16_t*>(slots + (c_now - first) % kNrSlots * kNrSlotBytes);
        const int h0 = (c_now - (kv ? cq : 0)) * kChunk + lane / LPH;
        Four x[kNrUnroll];
#pragma unroll
        for (int u = 0; u < kNrUnroll; ++u) {
          x[u] = {{0, 0}, {0, 0}};
          if (h0 + u * kHeads < n_heads && live) x[u] = load(chunk + (u * kHeads + lane / LPH) * p.dim);
        }
        __syncwarp();                                // the slot is read
        if (lane == 0 && c_now + kNrSlots < last) fetch(c_now + kNrSlots);
#pragma unroll
        for (int u = 0; u < kNrUnroll; ++u) {
          const int h = h0 + u * kHeads;
          uint64_t a[2], b[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            a[i] = widen<DT>(x[u].a[i]);
            b[i] = widen<DT>(x[u].b[i]);
          }
          float r = 1.f;
          if (norm) {
            uint64_t q = mul_f2(a[0], a[0]);
            q = fma_f2(b[0], b[0], q);
            q = fma_f2(a[1], a[1], q);
            q = fma_f2(b[1], b[1], q);
            float q0, q1;
            upk_f2(q, q0, q1);
            float ss = q0 + q1;
#pragma unroll
            for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor_sync(kAll, ss, o);
            r = rsqrtf(fmaf(ss, p.inv_dim, p.eps));
          }
          const uint64_t rr = pk_f2(r, r);
          Four z;
          if (REF) {
            Four y = x[u];
            if (norm) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                y.a[i] = Pk<DT>::mul(w.a[i], narrow<DT>(mul_f2(a[i], rr)));
                y.b[i] = Pk<DT>::mul(w.b[i], narrow<DT>(mul_f2(b[i], rr)));
              }
            }
            z = y;
            if (turns) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                z.a[i] = Pk<DT>::sub(Pk<DT>::mul(y.a[i], c16[i]), Pk<DT>::mul(y.b[i], s16[i]));
                z.b[i] = Pk<DT>::add(Pk<DT>::mul(y.b[i], c16[i]), Pk<DT>::mul(y.a[i], s16[i]));
              }
            }
          } else if (full) {                         // every lane turns: no selects (149 -> 141 us)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              z.a[i] = narrow<DT>(mul_f2(fma_f2(a[i], ca[i], mul_f2(b[i], sb[i])), rr));
              z.b[i] = narrow<DT>(mul_f2(fma_f2(b[i], cb[i], mul_f2(a[i], sa[i])), rr));
            }
          } else if (turns || norm) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              // (where nothing turns only the weight: 0 * x would spread a neighbour's infinity)
              const uint64_t za = turns ? fma_f2(a[i], ca[i], mul_f2(b[i], sb[i])) : mul_f2(a[i], ca[i]);
              const uint64_t zb = turns ? fma_f2(b[i], cb[i], mul_f2(a[i], sa[i])) : mul_f2(b[i], cb[i]);
              z.a[i] = narrow<DT>(mul_f2(za, rr));
              z.b[i] = narrow<DT>(mul_f2(zb, rr));
            }
          } else {
            z = x[u];
          }
          if (h < n_heads && live) store(dst + static_cast<int64_t>(h) * p.dim, z);
        }
      }
    }
  }
  for (; c_now < last && !failed; ++c_now) {
    if (!landed(c_now)) break;
    const int e0 = (c_now - cq - ck) * kVPiece;
    const uint16_t* chunk = reinterpret_cast<const uint16_t*>(slots + (c_now - first) % kNrSlots * kNrSlotBytes);
    uint4 x[kVPiece / 256];
#pragma unroll
    for (int i = 0; i < kVPiece / 256; ++i) x[i] = ld_vec(chunk + i * 256 + lane * 8);
    __syncwarp();
    if (lane == 0 && c_now + kNrSlots < last) fetch(c_now + kNrSlots);
#pragma unroll
    for (int i = 0; i < kVPiece / 256; ++i) {
      const int e = e0 + i * 256 + lane * 8;
      if (e < v_cols) st_vec(p.v_cache + row * p.kv_stride + e, x[i]);
    }
  }
  if (failed) {
    for (int c = c_now; c < min(last, c_now + kNrSlots); ++c) landed(c);
    report(p.status, CBK_STATUS_TIMEOUT);
  }
}

template <int DT, int LPH>
static int launch_norm_rope(NormRopeParams& p, int interleaved, int mode, cudaStream_t st) {
  constexpr int kHeads = 32 / LPH;
  constexpr int kChunk = kNrUnroll * kHeads, kVPiece = kNrSlotBytes / 2;
  const int chunks = (p.n_q + kChunk - 1) / kChunk + (p.n_kv + kChunk - 1) / kChunk +
                     (p.n_kv * p.dim + kVPiece - 1) / kVPiece;
  // a warp per token once that fills the GPU, else the chunks of a token over as many
  // warps as it takes
  const int64_t want = (kNrFill + p.n - 1) / p.n;
  p.parts = static_cast<int>(std::min<int64_t>(chunks, std::max<int64_t>(1, want)));
  const int64_t blocks = (p.n * p.parts + kNrWarps - 1) / kNrWarps;
  if (blocks > 0x7fffffff) return set_error(CBK_ERR_INVALID, "cbk_norm_rope_scatter: too many tokens");
  void (*kern)(const NormRopeParams) =
      mode == CBK_ROPE_REF ? (interleaved ? norm_rope_scatter_kernel<DT, LPH, true, true>
                                          : norm_rope_scatter_kernel<DT, LPH, true, false>)
                           : (interleaved ? norm_rope_scatter_kernel<DT, LPH, false, true>
                                          : norm_rope_scatter_kernel<DT, LPH, false, false>);
  if (int rc = ensure_smem_attr(reinterpret_cast<const void*>(kern), kNrSmem)) return rc;
  return launch_dependent("norm_rope_scatter_kernel", kern, dim3(static_cast<unsigned>(blocks)), dim3(kNrThreads), kNrSmem,
                          st, p);
}

template <int DT>
static int dispatch_norm_rope(NormRopeParams& p, int interleaved, int mode, cudaStream_t st) {
  if (p.dim <= 32) return launch_norm_rope<DT, 4>(p, interleaved, mode, st);
  if (p.dim <= 64) return launch_norm_rope<DT, 8>(p, interleaved, mode, st);
  if (p.dim <= 128) return launch_norm_rope<DT, 16>(p, interleaved, mode, st);
  return launch_norm_rope<DT, 32>(p, interleaved, mode, st);
}

}  // namespace cbk

using namespace cbk;

extern "C" int cbk_norm_rope_scatter(const cbk_norm_rope_scatter_args* a, void* stream) {
  if (!a || a->size != sizeof(*a)) return set_error(CBK_ERR_INVALID, "cbk_norm_rope_scatter: bad argument struct");
  const int dtype = a->dtype, head_dim = a->head_dim, rotary_dim = a->rotary_dim;
  if (dtype != CBK_BF16 && dtype != CBK_F16)
    return set_error(CBK_ERR_UNSUPPORTED, "cbk_norm_rope_scatter: dtype %d not supported", dtype);
  if (head_dim < 16 || head_dim > 256 || head_dim % 16 != 0)
    return set_error(CBK_ERR_UNSUPPORTED, "cbk_norm_rope_scatter: head_dim %d (multiples of 16 up to 256)", head_dim);
  if (rotary_dim < 16 || rotary_dim > head_dim || rotary_dim % 16 != 0)
    return set_error(CBK_ERR_UNSUPPORTED, "cbk_norm_rope_scatter: rotary_dim %d (multiples of 16 up to head_dim %d)",
                     rotary_dim, head_dim);
  if (a->rope_mode != CBK_ROPE_REF && a->rope_mode != CBK_ROPE_FP32)
    return set_error(CBK_ERR_INVALID, "cbk_norm_rope_scatter: rope_mode %d", a->rope_mode);
  if (a->n_q_heads <= 0 || a->n_kv_heads <= 0 || a->n_q_heads > 4096 || a->n_kv_heads > 4096)
    return set_error(CBK_ERR_INVALID, "cbk_norm_rope_scatter: bad head counts %d / %d", a->n_q_heads, a->n_kv_heads);
  if (a->n < 0 || a->cap < 0 || a->table_rows < 0)
    return set_error(CBK_ERR_INVALID, "cbk_norm_rope_scatter: negative size");
  if (a->n == 0) return CBK_OK;
  const int64_t qd = static_cast<int64_t>(a->n_q_heads) * head_dim, kd = static_cast<int64_t>(a->n_kv_heads) * head_dim;
  if (!a->q_src || !a->k_src || !a->v_src || !a->positions || !a->rows || !a->rope_table || !a->q_out ||
      !a->k_cache || !a->v_cache)
    return set_error(CBK_ERR_INVALID, "cbk_norm_rope_scatter: null pointer argument");
  if ((a->q_weight == nullptr) != (a->k_weight == nullptr))
    return set_error(CBK_ERR_INVALID, "cbk_norm_rope_scatter: give both weights or neither");
  if (a->q_row_stride < qd || a->k_row_stride < kd || a->v_row_stride < kd || a->kv_row_stride < kd ||
      (a->q_row_stride | a->k_row_stride | a->v_row_stride | a->kv_row_stride) % 8)
    return set_error(CBK_ERR_INVALID, "cbk_norm_rope_scatter: row strides must cover a row and be multiples of 8");
  const uintptr_t all = reinterpret_cast<uintptr_t>(a->q_src) | reinterpret_cast<uintptr_t>(a->k_src) |
                        reinterpret_cast<uintptr_t>(a->v_src) | reinterpret_cast<uintptr_t>(a->q_weight) |
                        reinterpret_cast<uintptr_t>(a->k_weight) | reinterpret_cast<uintptr_t>(a->rope_table) |
                        reinterpret_cast<uintptr_t>(a->q_out) | reinterpret_cast<uintptr_t>(a->k_cache) |
                        reinterpret_cast<uintptr_t>(a->v_cache);
  if (all & 15u) return set_error(CBK_ERR_INVALID, "cbk_norm_rope_scatter: pointers must be 16-byte aligned");
  NormRopeParams p;
  p.q = static_cast<const uint16_t*>(a->q_src);
  p.k = static_cast<const uint16_t*>(a->k_src);
  p.v = static_cast<const uint16_t*>(a->v_src);
  p.qw = static_cast<const uint16_t*>(a->q_weight);
  p.kw = static_cast<const uint16_t*>(a->k_weight);
  p.qs = a->q_row_stride;
  p.ks = a->k_row_stride;
  p.vs = a->v_row_stride;
  p.pos = a->positions;
  p.rows = a->rows;
  p.table = static_cast<const float4*>(a->rope_table);
  p.q_out = static_cast<uint16_t*>(a->q_out);
  p.k_cache = static_cast<uint16_t*>(a->k_cache);
  p.v_cache = static_cast<uint16_t*>(a->v_cache);
  p.status = a->status;
  p.n = a->n;
  p.table_rows = a->table_rows;
  p.cap = a->cap;
  p.kv_stride = a->kv_row_stride;
  p.n_q = a->n_q_heads;
  p.n_kv = a->n_kv_heads;
  p.dim = head_dim;
  p.rotary = rotary_dim;
  p.eps = a->eps;
  p.inv_dim = 1.f / static_cast<float>(head_dim);
  auto st = static_cast<cudaStream_t>(stream);
  return dtype == CBK_BF16 ? dispatch_norm_rope<CBK_BF16>(p, a->interleaved, a->rope_mode, st)
                           : dispatch_norm_rope<CBK_F16>(p, a->interleaved, a->rope_mode, st);
}

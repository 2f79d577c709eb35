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
// HBM-bound: every byte is read and written once.  A lane owns 8 consecutive
// elements (16 bytes) of a head, LPH = D / 8 rounded up to a power of two lanes
// make a head, a warp pass takes 32 / LPH heads, and a warp issues kUnroll
// passes' loads before any arithmetic.  The sum of squares is a butterfly within
// the head's lanes; the pair partner of the split layout lies R / 16 lanes away
// (R is a multiple of 16), so a shuffle brings it.  Everything is held in fp32;
// CBK_ROPE_REF adds the 16-bit roundings of the HF modules (the normalised value
// before and after its weight, cos and sin, each product and the sum), so the
// result has their bits; CBK_ROPE_FP32 rounds once, at the store.
#include "cbk_common.cuh"

namespace cbk {

constexpr int kNrThreads = 256;
constexpr int kNrWarps = kNrThreads / 32;
constexpr int kNrUnroll = 4;

struct NormRopeParams {
  const uint16_t *q, *k, *v, *qw, *kw;
  int64_t qs, ks, vs;             // source row strides
  const int64_t *pos, *rows;
  const float4* table;            // (cos, sin) pairs, two per float4
  uint16_t *q_out, *k_cache, *v_cache;
  int32_t* status;
  int64_t n, table_rows, cap, kv_stride;
  int n_q, n_kv, dim, rotary, chunks;   // chunks: warps per token
  float eps, inv_dim;
};

template <int DT, int LPH, bool REF, bool PAIRS>
__global__ void __launch_bounds__(kNrThreads)
norm_rope_scatter_kernel(const NormRopeParams p) {
  using E = Elem<DT>;
  constexpr int kHeads = 32 / LPH;          // heads per warp pass
  constexpr unsigned kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  const int64_t gw = static_cast<int64_t>(blockIdx.x) * kNrWarps + (threadIdx.x >> 5);
  const int64_t j = gw / p.chunks;
  if (j >= p.n) return;
  const int part = static_cast<int>(gw - j * p.chunks);
  const int64_t pos = p.pos[j], row = p.rows[j];
  const int l = lane & (LPH - 1), e0 = 8 * l;
  const int n_heads = p.n_q + 2 * p.n_kv;
  const int head0 = part * kNrUnroll * kHeads + lane / LPH;

  uint4 raw[kNrUnroll];
#pragma unroll
  for (int u = 0; u < kNrUnroll; ++u) {
    const int h = head0 + u * kHeads;
    raw[u] = make_uint4(0, 0, 0, 0);
    if (h < n_heads && e0 < p.dim) {
      const uint16_t* src;
      if (h < p.n_q) src = p.q + j * p.qs + static_cast<int64_t>(h) * p.dim;
      else if (h < p.n_q + p.n_kv) src = p.k + j * p.ks + static_cast<int64_t>(h - p.n_q) * p.dim;
      else src = p.v + j * p.vs + static_cast<int64_t>(h - p.n_q - p.n_kv) * p.dim;
      raw[u] = ld_stream(src + e0);
    }
  }
  if (row == -1) return;                    // padding token: nothing of it is written
  if (pos < 0 || pos >= p.table_rows || row < 0 || row >= p.cap) {
    if (part == 0 && lane == 0) report(p.status, CBK_STATUS_BAD_INDEX);
    return;
  }

  // cos / sin of the lane's elements: 8 pairs in the split layout, 4 interleaved
  constexpr int kCs = PAIRS ? 4 : 8;
  const bool turns = e0 < p.rotary;
  const int half = p.rotary / 2;
  float c[kCs], s[kCs];
  int partner = lane;
  {
    const int i0 = PAIRS ? e0 / 2 : (e0 < half ? e0 : e0 - half);
    const float4* t = p.table + (pos * half + i0) / 2;
#pragma unroll
    for (int i = 0; i < kCs / 2; ++i) {
      const float4 cs = turns ? __ldg(t + i) : make_float4(1.f, 0.f, 1.f, 0.f);
      c[2 * i] = cs.x;
      s[2 * i] = cs.y;
      c[2 * i + 1] = cs.z;
      s[2 * i + 1] = cs.w;
    }
    if (!PAIRS && turns) partner = e0 < half ? lane + half / 8 : lane - half / 8;
#pragma unroll
    for (int i = 0; i < kCs; ++i) {
      if (REF) {
        c[i] = round16<DT>(c[i]);
        s[i] = round16<DT>(s[i]);
      }
      if (!PAIRS && e0 < half) s[i] = -s[i];   // first of the pair: y_a c - y_b s
    }
  }
  const bool norm = p.qw != nullptr;
  uint4 wq = make_uint4(0, 0, 0, 0), wk = wq;
  if (norm && e0 < p.dim) {
    wq = ld_vec(p.qw + e0);
    wk = ld_vec(p.kw + e0);
  }

#pragma unroll
  for (int u = 0; u < kNrUnroll; ++u) {
    const int h = head0 + u * kHeads;
    const bool is_q = h < p.n_q, is_v = h >= p.n_q + p.n_kv;
    const uint16_t* hx = reinterpret_cast<const uint16_t*>(&raw[u]);
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = E::to_f(hx[e]);
    if (norm) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(y[e], y[e], ss);
#pragma unroll
      for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor_sync(kAll, ss, o);
      const float r = rsqrtf(fmaf(ss, p.inv_dim, p.eps));
      const uint4 w4 = is_q ? wq : wk;
      const uint16_t* hw = reinterpret_cast<const uint16_t*>(&w4);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float w = E::to_f(hw[e]);
        y[e] = REF ? round16<DT>(w * round16<DT>(y[e] * r)) : y[e] * r * w;
      }
    }
    float z[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (PAIRS) {
        const float other = y[e ^ 1], sn = (e & 1) ? s[e / 2] : -s[e / 2];
        z[e] = REF ? round16<DT>(y[e] * c[e / 2]) + round16<DT>(other * sn) : fmaf(y[e], c[e / 2], other * sn);
      } else {
        const float other = __shfl_sync(kAll, y[e], partner);
        z[e] = REF ? round16<DT>(y[e] * c[e % kCs]) + round16<DT>(other * s[e % kCs])
                   : fmaf(y[e], c[e % kCs], other * s[e % kCs]);
      }
    }
    if (h >= n_heads || e0 >= p.dim) continue;
    uint4 o = raw[u];
    if (!is_v) {
      uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = turns ? Pk<DT>::cvt(z[2 * e], z[2 * e + 1]) : Pk<DT>::cvt(y[2 * e], y[2 * e + 1]);
    }
    uint16_t* dst;
    if (is_q) dst = p.q_out + (j * p.n_q + h) * p.dim;
    else if (!is_v) dst = p.k_cache + row * p.kv_stride + static_cast<int64_t>(h - p.n_q) * p.dim;
    else dst = p.v_cache + row * p.kv_stride + static_cast<int64_t>(h - p.n_q - p.n_kv) * p.dim;
    st_vec(dst + e0, o);
  }
}

template <int DT, int LPH>
static int launch_norm_rope(NormRopeParams& p, int interleaved, int mode, cudaStream_t st) {
  constexpr int kHeads = 32 / LPH;
  const int passes = (p.n_q + 2 * p.n_kv + kHeads - 1) / kHeads;
  p.chunks = (passes + kNrUnroll - 1) / kNrUnroll;
  const int64_t blocks = (p.n * p.chunks + kNrWarps - 1) / kNrWarps;
  if (blocks > 0x7fffffff) return set_error(CBK_ERR_INVALID, "cbk_norm_rope_scatter: too many tokens");
  const unsigned g = static_cast<unsigned>(blocks);
  if (mode == CBK_ROPE_REF) {
    if (interleaved) norm_rope_scatter_kernel<DT, LPH, true, true><<<g, kNrThreads, 0, st>>>(p);
    else norm_rope_scatter_kernel<DT, LPH, true, false><<<g, kNrThreads, 0, st>>>(p);
  } else {
    if (interleaved) norm_rope_scatter_kernel<DT, LPH, false, true><<<g, kNrThreads, 0, st>>>(p);
    else norm_rope_scatter_kernel<DT, LPH, false, false><<<g, kNrThreads, 0, st>>>(p);
  }
  return check_launch("norm_rope_scatter_kernel");
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

// Attention of a tree of drafted tokens over the cache, on tcgen05 tensor cores.
//
// Node i of T nodes sees cache rows [0, n_ctx) and, of the rows n_ctx + j that
// hold the nodes' own K and V, those whose bit j is set in words[i]:
//   out[i][h] = softmax_t(scale q[i][h] . k[t][h / G]) . v[t][h / G].
// n_ctx is read on the device, so a captured step stays valid as it advances.
//
// The G q heads of a KV head share its keys, so the T * G query rows of a KV head
// (row = node * G + head) are stacked into Q tiles of 128 rows, and the keys are
// visited in tiles of 128.  The keys are split over CTAs -- grid (split, KV head,
// pair of Q tiles), about one CTA per SM -- and tree_merge_kernel joins the
// splits' (max, sum, O).  Up to 128 rows the call is bound by reading K and V
// once; beyond, a CTA runs two Q tiles on the same K and V.
//
// A CTA holds two "slots", each with S / P (128 columns) and O (HD columns) in
// TMEM and a softmax warpgroup of its own, so one slot's softmax runs while the
// tensor core works for the other.  With two Q tiles, slot t is tile t and every
// key tile goes to both; with one Q tile both slots hold that tile and take the
// key tiles in turn, each with its own running max, sum and O, joined at the end.
// Unit u of a CTA (slot u & 1) is then key tile u >> 1 or u, and the MMA warp's order
// is the same for both: O += P(u) V(u), then S(u + 2) = Q K(u + 2)^T, which overwrites
// P(u) after the PV that reads it.
//
// Warps (384 threads): 0 copies K and V tiles (TMA) into two rings; 1 issues the
// MMAs; 2 holds TMEM; 2 and 3 clean the V tiles that reach past the context; 4..7
// and 8..11 are the softmax of slots 0 and 1 (thread = row; a warp none of whose
// 32 rows exists takes no part, so small trees cost little).
//
// Masked keys: their scores become -inf in registers and their weight is 0
// exactly.  0 * NaN is NaN in an MMA, so rows behind the tree (whatever a cache
// holds there) are zeroed in the V tile, and so is every non-finite element of
// the tree's own V rows; the latter are added back on the CUDA cores, in the rows
// that see them, by the epilogue (only when there are any).
//
// Rounding: S, the softmax statistics, O, the partial results and the merge are
// fp32; P is rounded to the inputs' 16-bit type for the PV MMA (the tensor core
// takes both operands in one type), the result once.
//
// Visible keys: every exponential is ex2.approx, which keeps NaN and gives 0 for -inf.
// exp_chunk's polynomial for 3 of 16 pairs clamps its argument, so a NaN score would
// have weight 2^-126 there and an infinite one another than elsewhere.  Here the
// polynomial is slower too, since context and tree tiles would need code of their own
// (32 q heads on 8 KV heads of 128: 64 nodes over 32768 keys 43.3 us with it, 40.9
// without, 16 over 6208 13.4 and 13.2, 24 over 131072 90.8 and 90.9; 24 over 131072, 14
// on 2 heads of 64, 40.4 and 38.8).
//
// Measured, 32 q heads on 8 KV heads of 128, bf16, both kernels of the call: 24 nodes over
// 131072 keys 90 us (537 MB: 5.97 TB/s, 0.91 of measured HBM; 95 us in a long loop), 1
// node 86 us (6.2 TB/s);
// 64 nodes (two Q tiles) over 32768 keys 41 us (840 TFLOP/s with both products counted),
// over 16384 28.6: a key tile takes both slots 1.7 us, of which its bytes would take 1.44
// and its 32768 exponentials, 16 a clock, 1.04; 16 nodes over 6208 keys 13.1 us, 1 node
// 10.1 (HBM alone 3.9; traced at 10.8 us: set-up 1.5, key tiles 3.3, epilogue 1, merge
// launch and merge 3.5).
// Every wait is bounded; on timeout the kernel sets CBK_STATUS_TIMEOUT, drains its
// copies and MMAs, frees TMEM and returns.
#include <algorithm>
#include <type_traits>

#include "cbk_attn_common.cuh"

namespace cbk {

int ensure_smem_attr(const void* func, int bytes);   // cbk_api.cu

constexpr int kTreeThreads = 384;
constexpr int kTreeMaxNodes = 1024;
constexpr uint32_t kTreeTmemCols = 512;
constexpr int kTreeMergeWarps = 4;
constexpr int kTreeMaxSplits = 160;          // at most one per SM

struct TreeParams {
  const uint16_t *q, *v;
  const int64_t* n_ctx;
  const uint32_t* words;
  float* part_o;          // [slot][row_pitch][HD], relative to the slot's max
  float2* part_ml;        // [slot][row_pitch] (running max in log2 units, row sum)
  uint16_t* out;
  int32_t* status;
  int64_t kv_stride, words_stride, cap;
  int n_nodes, n_q, group, rows, n_qt, n_pairs, n_splits, row_pitch;
  float scale_log2;
};

// key tiles [j0, j1) of a split; tree-relative geometry of the call
struct TreeSpan {
  int64_t n_ctx, n_keys;
  int n_tiles;
  bool ok;
};
__device__ __forceinline__ TreeSpan tree_span(const TreeParams& p) {
  TreeSpan s;
  s.n_ctx = *p.n_ctx;
  s.ok = s.n_ctx >= 0 && s.n_ctx <= p.cap - p.n_nodes;
  s.n_keys = s.n_ctx + p.n_nodes;
  s.n_tiles = static_cast<int>((s.n_keys + kBN - 1) / kBN);
  return s;
}
// the first n_tiles % n_splits splits take one tile more than the others
__device__ __forceinline__ int split_start(int n_tiles, int n_splits, int s) {
  const int each = n_tiles / n_splits;
  return s * each + min(s, n_tiles - each * n_splits);
}

// 32 visibility bits of the keys at tree offsets [off, off + 32) of a node: offsets
// below 0 are context, those from n on are behind the tree
__device__ __forceinline__ uint32_t tree_bits(const uint32_t* w, int n, int off) {
  if (off <= -32) return 0xffffffffu;
  auto word = [&](int i) -> uint32_t {
    if (i * 32 >= n) return 0u;
    return n - i * 32 >= 32 ? w[i] : w[i] & ((1u << (n - i * 32)) - 1u);
  };
  if (off < 0) return ((1u << -off) - 1u) | (word(0) << -off);
  return __funnelshift_r(word(off >> 5), word((off >> 5) + 1), off & 31);
}

// 1 / l of a row; without any weight 0, or NaN (the formula's 0 / 0) when the row sees
// keys after all, each with a score of -inf
__device__ __forceinline__ float tree_inverse(const TreeParams& p, int64_t n_ctx, int node, float l) {
  if (l != 0.f) return 1.f / l;
  bool sees = n_ctx > 0;
  for (int off = 0; off < p.n_nodes && !sees; off += 32)
    sees = tree_bits(p.words + node * p.words_stride, p.n_nodes, off) != 0;
  return sees ? __int_as_float(0x7fffffff) : 0.f;
}

// 16 bytes from global to shared memory, asynchronously; zeros when not `there`
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

template <int HD, int NQ>
struct TreeSmem {
  // K and V tiles in flight.  One Q tile, 32 q heads on 8 KV heads of 128: 3 against 2 is
  // 90.9 against 91.6 us for 24 nodes over 131072 keys, 10.1 against 10.2 for 1 over 6208,
  // but 13.2 against 12.4 for 16 over 6208; 14 on 2 heads of 64, 24 over 131072: 39.5 with
  // 2, 38.8 with 3 and with 4, 38.9 with 6.  Two Q tiles: 3 do not fit with heads of 128;
  // 32 on 8 heads of 64, 64 over 16384: 24.3 to 26.6 with 2, 3 and 5, no order among them.
  static constexpr int kStages = NQ == 1 ? 3 : 2;
  static constexpr int kQBytes = kBM * HD * 2;
  static constexpr int kKVBytes = kBN * HD * 2;
  static constexpr int kK0 = NQ * kQBytes;
  static constexpr int kV0 = kK0 + kStages * kKVBytes;
  static constexpr int kBar = kV0 + kStages * kKVBytes;
  static constexpr int kBars = 5 * kStages + 9;
  static constexpr int kMisc = kBar + kBars * 8;       // tmem slot, abort flag, non-finite flag
  static constexpr int kTotal = kMisc + 16;
  // more than half an SM's shared memory: one CTA (holding all 512 TMEM columns) per SM
  static constexpr int kAlloc = (kTotal + 1024) > 122880 ? (kTotal + 1024) : 122880;
};

template <int DT, int HD, int NQ>
__global__ void __launch_bounds__(kTreeThreads, 1)
tree_attn_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                 const TreeParams p) {
  using L = TreeSmem<HD, NQ>;
  constexpr int NST = L::kStages;
  enum { KFULL = 0, KEMPTY = NST, VFULL = 2 * NST, VEMPTY = 3 * NST, VCLEAN = 4 * NST, SFULL = 5 * NST,
         PHALF = SFULL + 2, PFULL = SFULL + 4, ODONE = SFULL + 6, DRAIN = SFULL + 8 };
  const int split = blockIdx.x, kvh = blockIdx.y, pair = blockIdx.z;
  grid_wait();
  const TreeSpan sp = tree_span(p);
  if (!sp.ok) {
    if (threadIdx.x == 0 && split == 0 && kvh == 0 && pair == 0) report(p.status, CBK_STATUS_BAD_INDEX);
    return;
  }
  const int j0 = split_start(sp.n_tiles, p.n_splits, split);
  const int n = split_start(sp.n_tiles, p.n_splits, split + 1) - j0;      // key tiles of this CTA
  if (n == 0) return;
  const bool two = NQ == 2 && 2 * pair + 1 < p.n_qt;       // two Q tiles, else one in both slots
  const int n_units = two ? 2 * n : n;
  // first local key tile that is not all context
  const int n_full = static_cast<int>(sp.n_ctx / kBN);
  const int m0 = n_full > j0 ? min(n_full - j0, n) : 0;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t* sbase = smem_raw + (base - raw_addr);
  const uint32_t sK0 = base + L::kK0, sV0 = base + L::kV0;
  auto bar = [&](int i) { return base + L::kBar + 8u * i; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sbase + L::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sbase + L::kMisc + 4);
  volatile int* odd_flag = reinterpret_cast<volatile int*>(sbase + L::kMisc + 8);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  bool failed = false;
  auto wait_all = [&](uint32_t b, uint32_t parity) {
    return __all_sync(0xffffffffu, wait_or_abort(b, parity, abort_flag));
  };
  auto tile_rows = [&](int t) {                  // existing rows of slot t's Q tile
    return min(kBM, p.rows - (2 * pair + (two ? t : 0)) * kBM);
  };
  auto load_tile = [&](const CUtensorMap* tm, uint32_t dst, uint32_t b, int g) {
    mbar_expect_tx(b, L::kKVBytes);
#pragma unroll
    for (int h = 0; h < HD / 64; ++h) tma_load_3d(dst + h * (kBN * 128), tm, b, h * 64, kvh, (j0 + g) * kBN);
  };

  if (warp == 0) {
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < NST; ++i) {
        mbar_init(bar(KFULL + i), 1);
        mbar_init(bar(KEMPTY + i), 1);
        mbar_init(bar(VFULL + i), 1);
        mbar_init(bar(VEMPTY + i), 3);           // the MMAs' commit and the two cleaning warps
        mbar_init(bar(VCLEAN + i), 2);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int active = (tile_rows(t) + 31) / 32;
        mbar_init(bar(SFULL + t), 1);
        mbar_init(bar(PHALF + t), active);
        mbar_init(bar(PFULL + t), active);
        mbar_init(bar(ODONE + t), 1);
      }
      mbar_init(bar(DRAIN), 1);
      *abort_flag = 0;
      *odd_flag = 0;
      fence_barrier_init();
    }
    __syncwarp();
    if (elect_one()) {                           // the first tiles are on their way before the rest is set up
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      for (int g = 0; g < min(n, NST); ++g) {
        load_tile(&tm_k, sK0 + g * L::kKVBytes, bar(KFULL + g), g);
        load_tile(&tm_v, sV0 + g * L::kKVBytes, bar(VFULL + g), g);
      }
    }
  } else if (warp == 2) {
    tmem_alloc(smem_u32(tmem_slot), kTreeTmemCols);
    tmem_relinquish();
  } else if (warp >= 4) {
    // Q tiles in the layout a 128-byte-swizzled TMA copy leaves: 16-byte piece c of
    // row r at piece c ^ (r & 7); rows that do not exist are zero
    constexpr int kVec = HD / 8, kStep = (kTreeThreads - 128) / kVec;
    const int c = threadIdx.x % kVec, row0 = 2 * pair * kBM;
    const int n_rows = (two ? 2 : 1) * kBM;
#pragma unroll 8
    for (int r = (threadIdx.x - 128) / kVec; r < n_rows; r += kStep) {
      const int row = min(row0 + r, p.rows - 1), node = row / p.group;
      cp_async16_or_zero(base + (r / kBM) * L::kQBytes + (c >> 3) * (kBM * 128) + (r % kBM) * 128 + ((c ^ r) & 7) * 16,
                         p.q + (static_cast<int64_t>(node) * p.n_q + kvh * p.group + row - node * p.group) * HD + c * 8,
                         row0 + r < p.rows);
    }
    asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // the merge kernel (a programmatic dependent) may be placed as SMs free up
  grid_launch_dependents();

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    const bool leader = elect_one();
    int last_k = min(n, NST) - 1, last_v = last_k;      // last tiles issued
    for (int g = NST; g < n; ++g) {
      const int st = g % NST;
      const uint32_t par = (g / NST - 1) & 1;
      if (!wait_all(bar(KEMPTY + st), par)) {
        failed = true;
        break;
      }
      if (leader) load_tile(&tm_k, sK0 + st * L::kKVBytes, bar(KFULL + st), g);
      last_k = g;
      if (!wait_all(bar(VEMPTY + st), par)) {
        failed = true;
        break;
      }
      if (leader) load_tile(&tm_v, sV0 + st * L::kKVBytes, bar(VFULL + st), g);
      last_v = g;
    }
    // drain: every armed copy must land before the CTA can retire
    for (int g = max(0, last_k - NST + 1); g <= last_k; ++g)
      if (!__all_sync(0xffffffffu, mbar_wait(bar(KFULL + g % NST), (g / NST) & 1))) failed = true;
    for (int g = max(0, last_v - NST + 1); g <= last_v; ++g)
      if (!__all_sync(0xffffffffu, mbar_wait(bar(VFULL + g % NST), (g / NST) & 1))) failed = true;
  } else if (warp == 1) {
    // ------------------------------------------------------------- MMA issuer
    const bool leader = elect_one();
    const uint32_t idesc_s = umma_idesc_f16(DT, kBM, kBN, 0);
    const uint32_t idesc_o = umma_idesc_f16(DT, kBM, HD, 1);
    const uint64_t dq0 = umma_desc_sw128(base, 16, 1024);
    const uint64_t dk0 = umma_desc_sw128(sK0, 16, 1024);
    const uint64_t dv0 = umma_desc_sw128(sV0, kBN * 128, 1024);
    auto unit_tile = [&](int u) { return two ? u >> 1 : u; };
    // S of unit u, waiting for its K tile at the tile's first use and releasing it after its last
    auto issue_s = [&](int u) -> bool {
      const int t = u & 1, g = unit_tile(u), st = g % NST;
      if (!(two && t == 1) && !wait_all(bar(KFULL + st), (g / NST) & 1)) return false;
      tc_fence_after();
      const uint64_t q0 = dq0 + ((two && t) ? (L::kQBytes >> 4) : 0);
      const uint64_t k0 = dk0 + ((st * L::kKVBytes) >> 4);
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        const uint32_t off = ((kk >> 2) * (kBM * 128) + (kk & 3) * 32) >> 4;
        if (leader) umma_f16_ss(tmem + 256 * t, q0 + off, k0 + off, idesc_s, kk > 0 ? 1u : 0u);
      }
      if (leader) {
        umma_commit(bar(SFULL + t));
        if (!two || t == 1) umma_commit(bar(KEMPTY + st));
      }
      return true;
    };
    auto issue_pv = [&](int t, int st, bool acc, int kk_lo, int kk_hi) {
      const uint64_t v0 = dv0 + ((st * L::kKVBytes) >> 4);
#pragma unroll
      for (int kk = kk_lo; kk < kk_hi; ++kk)
        if (leader)
          umma_f16_ts(tmem + 256 * t + kBN, tmem + 256 * t + kk * 8, v0 + ((kk * 16 * 128) >> 4), idesc_o,
                      (acc || kk > 0) ? 1u : 0u);
    };
    for (int u = 0; u < min(n_units, 2) && !failed; ++u)
      if (!issue_s(u)) failed = true;
    for (int u = 0; u < n_units && !failed; ++u) {
      const int t = u & 1, g = unit_tile(u), st = g % NST, k = u >> 1;     // unit k of its slot
      if (!(two && t == 1)) {
        const bool ok = g < m0 ? wait_all(bar(VFULL + st), (g / NST) & 1)
                               : wait_all(bar(VCLEAN + st), ((g - m0) / NST) & 1);
        if (!ok) {
          failed = true;
          break;
        }
      }
      if (!wait_all(bar(PHALF + t), k & 1)) {
        failed = true;
        break;
      }
      tc_fence_after();
      issue_pv(t, st, k > 0, 0, kBN / 32);
      if (!wait_all(bar(PFULL + t), k & 1)) {
        failed = true;
        break;
      }
      tc_fence_after();
      issue_pv(t, st, true, kBN / 32, kBN / 16);
      if (leader && (!two || t == 1)) umma_commit(bar(VEMPTY + st));
      if (u + 2 < n_units) {
        if (!issue_s(u + 2)) failed = true;
      } else if (leader) {
        umma_commit(bar(ODONE + t));
      }
    }
    // drain: all MMAs issued by this warp complete before TMEM is released
    if (leader) umma_commit(bar(DRAIN));
    if (!__all_sync(0xffffffffu, mbar_wait(bar(DRAIN), 0))) failed = true;
  } else if (warp < 4) {
    // -------------------------------------- V tiles that reach past the context
    constexpr uint32_t kExp = DT == CBK_BF16 ? 0x7f80u : 0x7c00u;
    // Tiles of context pass through: these warps see every phase of every stage, and a
    // stage is filled again only once they have left it.
    for (int g = 0; g < n; ++g) {
      const int st = g % NST;
      if (!wait_all(bar(VFULL + st), (g / NST) & 1)) {
        failed = true;
        break;
      }
      if (g < m0) {
        if (lane == 0) mbar_arrive(bar(VEMPTY + st));
        continue;
      }
      const int64_t t0 = static_cast<int64_t>(j0 + g) * kBN;
      const int tree0 = static_cast<int>(sp.n_ctx > t0 ? sp.n_ctx - t0 : 0);                  // first row of the tree
      const int end = static_cast<int>(min(static_cast<int64_t>(kBN), sp.n_keys - t0));       // first row behind it
      uint4* tile = reinterpret_cast<uint4*>(sbase + L::kV0 + st * L::kKVBytes);
      bool odd = false;
      for (int i = threadIdx.x - 64; i < L::kKVBytes / 16; i += 64) {
        const int r = (i >> 3) % kBN;
        if (r < tree0) continue;
        uint4 x = tile[i];
        uint32_t* w = reinterpret_cast<uint32_t*>(&x);
        if (r >= end) {
          tile[i] = make_uint4(0, 0, 0, 0);
          continue;
        }
        bool here = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if ((w[e] & kExp) == kExp) w[e] &= 0xffff0000u, here = true;
          if ((w[e] & (kExp << 16)) == (kExp << 16)) w[e] &= 0x0000ffffu, here = true;
        }
        if (here) {
          tile[i] = x;
          odd = true;
        }
      }
      if (odd) *odd_flag = 1;
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar(VCLEAN + st));
        mbar_arrive(bar(VEMPTY + st));
      }
    }
  } else {
    // ----------------------------------------------- softmax + epilogue warps
    const int t = (warp - 4) >> 2, sub = warp & 3;
    const int row = sub * 32 + lane;                        // row of the Q tile
    const int n_rows = tile_rows(t);
    const int n_t = two ? n : (n - t + 1) / 2;              // units of this slot
    if (sub * 32 < n_rows && n_t > 0) {
      const uint32_t lane_off = static_cast<uint32_t>(sub * 32) << 16;
      const uint32_t tS = tmem + 256 * t + lane_off, tO = tS + kBN;
      const float sl2 = p.scale_log2;
      const int node = min((2 * pair + (two ? t : 0)) * kBM + row, p.rows - 1) / p.group;
      const uint32_t* words = p.words + node * p.words_stride;
      float m_used = -INFINITY, l_sum = 0.f;
      for (int k = 0; k < n_t; ++k) {
        const int g = two ? k : 2 * k + t;
        if (!wait_all(bar(SFULL + t), k & 1)) {
          failed = true;
          break;
        }
        tc_fence_after();
        uint32_t s[kBN];
#pragma unroll
        for (int c4 = 0; c4 < kBN / 32; ++c4) tmem_ld32(tS + c4 * 32, *reinterpret_cast<uint32_t(*)[32]>(&s[c4 * 32]));
        tmem_wait_ld();
        const bool masked = g >= m0;
        if (masked) {
          const int off = static_cast<int>(static_cast<int64_t>(j0 + g) * kBN - sp.n_ctx);
#pragma unroll
          for (int c4 = 0; c4 < kBN / 32; ++c4) {
            const uint32_t bits = tree_bits(words, p.n_nodes, off + 32 * c4);
#pragma unroll
            for (int e = 0; e < 32; ++e) s[c4 * 32 + e] = (bits >> e) & 1u ? s[c4 * 32 + e] : 0xff800000u;
          }
        }
        float x0 = -INFINITY, x1 = -INFINITY, x2 = -INFINITY, x3 = -INFINITY;
#pragma unroll
        for (int c = 0; c < kBN; c += 8) {
          x0 = max3f(x0, __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
          x1 = max3f(x1, __uint_as_float(s[c + 2]), __uint_as_float(s[c + 3]));
          x2 = max3f(x2, __uint_as_float(s[c + 4]), __uint_as_float(s[c + 5]));
          x3 = max3f(x3, __uint_as_float(s[c + 6]), __uint_as_float(s[c + 7]));
        }
        const float m_tile = max3f(x0, x1, fmaxf(x2, x3)) * sl2;
        float alpha = 1.f;
        bool rescale = false;
        if (k == 0) {
          m_used = m_tile;
        } else if (m_tile > m_used + 8.f) {      // P stays below 2^8 under the older max
          alpha = ex2(m_used - m_tile);
          m_used = m_tile;
          rescale = true;
        }
        float ra0 = 0.f, ra1 = 0.f, rb0 = 0.f, rb1 = 0.f;
        // no visible key so far: a finite offset keeps the masked arguments at -inf
        const float neg_m = m_used == -INFINITY ? 0.f : -m_used;
#pragma unroll
        for (int c4 = 0; c4 < kBN / 32; ++c4) {
          uint32_t pk[16];
          exp_chunk<DT, 0>(s, c4, sl2, neg_m, ra0, ra1, rb0, rb1, pk);
          tmem_st16(tS + c4 * 16, pk);
          if (c4 == kBN / 64 - 1) {
            // keys 0-63 of P stored: their PV may start, once O has the new max (O is
            // stable: the commit behind this tile's S covered the PV before it)
            if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
              for (int c = 0; c < HD / 32; ++c) {
                uint32_t o[32];
                tmem_ld32(tO + c * 32, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                tmem_st32(tO + c * 32, o);
              }
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(PHALF + t));
          }
        }
        l_sum = l_sum * alpha + (ra0 + ra1) + (rb0 + rb1);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(PFULL + t));
      }
      // One Q tile: both slots' O lie in the same TMEM lanes, so the two warps of a
      // row join them, each for half of the head dimensions.  Two: every slot is its
      // tile's result.
      const bool other = !two && n > 1;                      // the other slot holds a part of this row
      if (!failed && !wait_all(bar(ODONE + t), 0)) failed = true;
      if (!failed && other && !wait_all(bar(ODONE + (t ^ 1)), 0)) failed = true;
      float w_own = 1.f, w_other = 0.f;
      if (other) {
        // (every MMA is complete: Q's room is free for the rows' (max, sum))
        float2* ml = reinterpret_cast<float2*>(sbase);
        ml[t * kBM + row] = make_float2(m_used, l_sum);
        // the active warps of both slots (a warp that failed arrives too)
        asm volatile("bar.sync 1, %0;" ::"r"(2 * 32 * ((n_rows + 31) / 32)) : "memory");
        const float2 x = ml[(t ^ 1) * kBM + row];
        // a slot without a visible key has l = 0 and weight 0; its O is 0
        const float m = fmaxf(l_sum != 0.f ? m_used : -INFINITY, x.y != 0.f ? x.x : -INFINITY);
        w_own = l_sum != 0.f ? ex2(m_used - m) : 0.f;
        w_other = x.y != 0.f ? ex2(x.x - m) : 0.f;
        l_sum = (l_sum != 0.f ? w_own * l_sum : 0.f) + (x.y != 0.f ? w_other * x.y : 0.f);
        m_used = m;
      }
      if (!failed) {
        tc_fence_after();
        const bool direct = min(sp.n_tiles, p.n_splits) == 1;          // this CTA alone has the row's keys
        const int64_t slot = ((static_cast<int64_t>(kvh) * p.n_pairs + pair) * p.n_splits + split) * NQ + (two ? t : 0);
        float* po = p.part_o + (slot * p.row_pitch + row) * HD;
        const int grow = (2 * pair + (two ? t : 0)) * kBM + row;
        uint16_t* out = p.out + (static_cast<int64_t>(node) * p.n_q + kvh * p.group + grow % p.group) * HD;
        const float inv = direct ? tree_inverse(p, sp.n_ctx, node, l_sum) : 1.f;
        const bool fix = *odd_flag != 0;
        const uint32_t t_other = tmem + 256 * (t ^ 1) + lane_off + kBN;
        // columns of 32: this warp's share
        const int c_lo = other && t == 1 ? HD / 64 : 0, c_hi = other && t == 0 ? HD / 64 : HD / 32;
        for (int c = c_lo; c < c_hi; ++c) {
          uint32_t o[32];
          tmem_ld32(tO + c * 32, o);
          if (other) {
            uint32_t y[32];
            tmem_ld32(t_other + c * 32, y);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e)
              o[e] = __float_as_uint(__uint_as_float(o[e]) * w_own + __uint_as_float(y[e]) * w_other);
          } else {
            tmem_wait_ld();
          }
          if (row < n_rows && fix) {
            // non-finite elements of the V rows this row sees in this CTA's key tiles
            for (int g = m0; g < n; ++g) {
              const int off = static_cast<int>(static_cast<int64_t>(j0 + g) * kBN - sp.n_ctx);
              for (int b = max(0, -off); b < kBN && off + b < p.n_nodes; ++b) {
                const int j = off + b;
                if (!((words[j >> 5] >> (j & 31)) & 1u)) continue;
                const uint16_t* vr = p.v + (sp.n_ctx + j) * p.kv_stride + static_cast<int64_t>(kvh) * HD + c * 32;
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  const float x = Elem<DT>::to_f(vr[e]);
                  if (!(fabsf(x) < INFINITY)) o[e] = __float_as_uint(__uint_as_float(o[e]) + x);
                }
              }
            }
          }
          if (row < n_rows) {
            if (direct) {
              store_chunk<DT>(out + c * 32, o, inv, false);
            } else {
#pragma unroll
              for (int h = 0; h < 4; ++h)
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                             :: "l"(po + c * 32 + 8 * h), "r"(o[8 * h]), "r"(o[8 * h + 1]), "r"(o[8 * h + 2]),
                                "r"(o[8 * h + 3]), "r"(o[8 * h + 4]), "r"(o[8 * h + 5]), "r"(o[8 * h + 6]),
                                "r"(o[8 * h + 7]) : "memory");
            }
          }
          __syncwarp();
        }
        if (row < n_rows && !direct && (two || t == 0)) p.part_ml[slot * p.row_pitch + row] = make_float2(m_used, l_sum);
      }
    }
  }

  if (failed) {
    *abort_flag = 1;
    report(p.status, CBK_STATUS_TIMEOUT);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, kTreeTmemCols);
  }
}

// Merge of the splits, a warp per query row: O = sum_i w_i O_i / sum_i w_i l_i,
// w_i = 2^(m_i - M) over the splits that hold a key tile, in their order, sixteen O
// loads in flight (behind branches, one by one: 24 us instead of 10 for 64 nodes over
// 32768 keys, 19 MB of partial results).  A row that sees nothing has every l_i = 0.
// (With one such split the attention kernel has written the output.)
template <int DT, int HD>
__global__ void __launch_bounds__(kTreeMergeWarps * 32)
tree_merge_kernel(const TreeParams p, int n_kv) {
  constexpr int kD = HD / 32, kAhead = 16;
  using Vec = typename std::conditional<kD == 4, float4, float2>::type;
  __shared__ float s_w[kTreeMergeWarps][kTreeMaxSplits];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t gr = static_cast<int64_t>(blockIdx.x) * kTreeMergeWarps + warp;
  if (gr >= static_cast<int64_t>(n_kv) * p.rows) return;
  const int kvh = static_cast<int>(gr / p.rows), row = static_cast<int>(gr % p.rows);
  const int qt = row / kBM, pair = qt / 2, r = row % kBM;
  const int per = p.n_qt == 1 ? 1 : 2;                 // slots of a split
  const int64_t slot0 = (static_cast<int64_t>(kvh) * p.n_pairs + pair) * p.n_splits * per +
                        ((qt | 1) < p.n_qt ? qt & 1 : 0);
  const float2* ml = p.part_ml + slot0 * p.row_pitch + r;
  const float* po = p.part_o + (slot0 * p.row_pitch + r) * HD + lane * kD;
  const int64_t step = static_cast<int64_t>(per) * p.row_pitch;
  // (n_ctx is no result of the attention kernel, which began once its writer was done)
  const TreeSpan sp = tree_span(p);
  grid_wait();
  grid_launch_dependents();
  if (!sp.ok) return;                                  // reported by the attention kernel
  const int n = min(sp.n_tiles, p.n_splits);           // splits 0 .. n - 1 hold key tiles
  if (n == 1) return;
  Vec x[kAhead];
  auto load = [&](int i0) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (i0 + k < n) x[k] = *reinterpret_cast<const Vec*>(po + (i0 + k) * step * HD);
  };
  load(0);                                             // on its way beside the (m, l) pairs
  float2 mine[kTreeMaxSplits / 32];
  float M = -INFINITY;
#pragma unroll
  for (int q = 0; q < kTreeMaxSplits / 32; ++q) {
    mine[q] = lane + 32 * q < n ? ml[(lane + 32 * q) * step] : make_float2(-INFINITY, 0.f);
    if (mine[q].y != 0.f) M = fmaxf(M, mine[q].x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  float lsum = 0.f;
#pragma unroll
  for (int q = 0; q < kTreeMaxSplits / 32; ++q) {
    const float w = mine[q].y != 0.f ? ex2(mine[q].x - M) : 0.f;
    s_w[warp][lane + 32 * q] = w;
    lsum += mine[q].y != 0.f ? w * mine[q].y : 0.f;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) lsum += __shfl_xor_sync(0xffffffffu, lsum, o);
  __syncwarp();
  float acc[kD];
#pragma unroll
  for (int d = 0; d < kD; ++d) acc[d] = 0.f;
  for (int i0 = 0; i0 < n; i0 += kAhead) {
    if (i0 > 0) load(i0);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (i0 + k >= n) break;
      const float w = s_w[warp][i0 + k];
      acc[0] = fmaf(w, x[k].x, acc[0]);
      acc[1] = fmaf(w, x[k].y, acc[1]);
      if constexpr (kD == 4) {
        acc[2] = fmaf(w, x[k].z, acc[2]);
        acc[3] = fmaf(w, x[k].w, acc[3]);
      }
    }
  }
  const float inv = tree_inverse(p, sp.n_ctx, row / p.group, lsum);
  uint16_t* o = p.out + (static_cast<int64_t>(row / p.group) * p.n_q + kvh * p.group + row % p.group) * HD + lane * kD;
#pragma unroll
  for (int d = 0; d < kD; d += 2) *reinterpret_cast<uint32_t*>(o + d) = Pk<DT>::cvt(acc[d] * inv, acc[d + 1] * inv);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct TreeLayout {
  int rows, n_qt, n_pairs, n_splits, row_pitch;
  size_t off_o, bytes;
};

static TreeLayout tree_layout(int n_nodes, int64_t cap, int n_q_heads, int n_kv_heads, int head_dim) {
  TreeLayout t;
  t.rows = n_nodes * (n_q_heads / n_kv_heads);
  t.n_qt = (t.rows + kBM - 1) / kBM;
  t.n_pairs = (t.n_qt + 1) / 2;
  const int64_t units = static_cast<int64_t>(n_kv_heads) * t.n_pairs;
  const int64_t sms = std::min(attn_sm_count(), kTreeMaxSplits);
  t.n_splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sms / units, (cap + kBN - 1) / kBN)));
  t.row_pitch = (std::min(t.rows, kBM) + 7) / 8 * 8;
  // one split writes the output itself
  const size_t slots = t.n_splits == 1 ? 0 : static_cast<size_t>(units) * t.n_splits * (t.n_qt == 1 ? 1 : 2);
  t.off_o = (slots * t.row_pitch * sizeof(float2) + 255) & ~static_cast<size_t>(255);
  t.bytes = std::max<size_t>(256, t.off_o + slots * t.row_pitch * head_dim * sizeof(float));
  return t;
}

template <int DT, int HD, int NQ>
static int launch_tree(const cbk_tree_attn_args* a, const TreeParams& p, cudaStream_t st) {
  CUtensorMap mk, mv;
  if (int rc = attn_make_map(&mk, a->k_cache, DT, HD, a->n_kv_heads, a->cap, a->kv_row_stride, 1, kBN)) return rc;
  if (int rc = attn_make_map(&mv, a->v_cache, DT, HD, a->n_kv_heads, a->cap, a->kv_row_stride, 1, kBN)) return rc;
  auto kern = tree_attn_kernel<DT, HD, NQ>;
  constexpr int smem = TreeSmem<HD, NQ>::kAlloc;
  static_assert(smem <= 227 * 1024, "shared memory of tree_attn_kernel");
  if (int rc = ensure_smem_attr(reinterpret_cast<const void*>(kern), smem)) return rc;
  if (int rc = launch_dependent("tree_attn_kernel", kern, dim3(p.n_splits, a->n_kv_heads, p.n_pairs),
                                dim3(kTreeThreads), smem, st, mk, mv, p))
    return rc;
  if (p.n_splits == 1) return CBK_OK;
  const int64_t rows = static_cast<int64_t>(a->n_kv_heads) * p.rows;
  return launch_dependent("tree_merge_kernel", tree_merge_kernel<DT, HD>,
                          dim3(static_cast<unsigned>((rows + kTreeMergeWarps - 1) / kTreeMergeWarps)),
                          dim3(kTreeMergeWarps * 32), 0, st, p, static_cast<int>(a->n_kv_heads));
}

template <int DT>
static int dispatch_tree(const cbk_tree_attn_args* a, const TreeParams& p, cudaStream_t st) {
  // One Q tile in both slots or two: the first could run as the second with one tile,
  // but takes half the workspace and has room for a third stage (24 nodes over 131072
  // keys, 14 on 2 heads of 64: 38.8 us against 39.2; 37 over 1029, 4 on 2 heads of 64, 7.1
  // against 7.4; 24 over 131072, 32 on 8 heads of 128, 90.9 against 90.6; 16 over 6208,
  // which likes two stages better, 13.2 against 12.4).
  if (a->head_dim == 128) return p.n_qt == 1 ? launch_tree<DT, 128, 1>(a, p, st) : launch_tree<DT, 128, 2>(a, p, st);
  return p.n_qt == 1 ? launch_tree<DT, 64, 1>(a, p, st) : launch_tree<DT, 64, 2>(a, p, st);
}

}  // namespace cbk

using namespace cbk;

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
  return tree_layout(std::max(n_nodes, 1), std::max<int64_t>(cap, 1), n_q_heads, n_kv_heads, head_dim).bytes;
}

extern "C" int cbk_tree_attn(const cbk_tree_attn_args* a, void* stream) {
  if (!a || a->size != sizeof(*a)) return set_error(CBK_ERR_INVALID, "cbk_tree_attn: bad argument struct");
  if (a->dtype != CBK_BF16 && a->dtype != CBK_F16)
    return set_error(CBK_ERR_UNSUPPORTED, "cbk_tree_attn: dtype %d not supported", a->dtype);
  if (int rc = check_tree_geometry("cbk_tree_attn", a->n_nodes, a->cap, a->n_q_heads, a->n_kv_heads, a->head_dim))
    return rc;
  if (a->n_nodes == 0) return CBK_OK;
  if (a->kv_row_stride < static_cast<int64_t>(a->n_kv_heads) * a->head_dim || a->kv_row_stride % 8 != 0 ||
      a->words_stride < (a->n_nodes + 31) / 32)
    return set_error(CBK_ERR_INVALID, "cbk_tree_attn: bad strides (cache %lld, words %lld)",
                     (long long)a->kv_row_stride, (long long)a->words_stride);
  if (!a->q || !a->k_cache || !a->v_cache || !a->n_ctx || !a->words || !a->out || !a->workspace)
    return set_error(CBK_ERR_INVALID, "cbk_tree_attn: null pointer argument");
  if (reinterpret_cast<uintptr_t>(a->workspace) & 31u)
    return set_error(CBK_ERR_INVALID, "cbk_tree_attn: the workspace must be 32-byte aligned");
  if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k_cache) |
       reinterpret_cast<uintptr_t>(a->v_cache) | reinterpret_cast<uintptr_t>(a->out)) & 15u)
    return set_error(CBK_ERR_INVALID, "cbk_tree_attn: q, caches and out must be 16-byte aligned");
  if (!(a->scale > 0.f) || !(a->scale < INFINITY))
    return set_error(CBK_ERR_INVALID, "cbk_tree_attn: scale must be positive and finite");
  const TreeLayout lay = tree_layout(a->n_nodes, a->cap, a->n_q_heads, a->n_kv_heads, a->head_dim);
  if (lay.n_pairs > 65535 || a->n_kv_heads > 65535)
    return set_error(CBK_ERR_UNSUPPORTED, "cbk_tree_attn: too many query rows");
  if (a->workspace_bytes < 0 || static_cast<size_t>(a->workspace_bytes) < lay.bytes)
    return set_error(CBK_ERR_WORKSPACE, "cbk_tree_attn: workspace %lld < %zu bytes", (long long)a->workspace_bytes,
                     lay.bytes);
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  TreeParams p;
  p.q = static_cast<const uint16_t*>(a->q);
  p.v = static_cast<const uint16_t*>(a->v_cache);
  p.n_ctx = a->n_ctx;
  p.words = reinterpret_cast<const uint32_t*>(a->words);
  p.part_ml = reinterpret_cast<float2*>(ws);
  p.part_o = reinterpret_cast<float*>(ws + lay.off_o);
  p.out = static_cast<uint16_t*>(a->out);
  p.status = a->status;
  p.kv_stride = a->kv_row_stride;
  p.words_stride = a->words_stride;
  p.cap = a->cap;
  p.n_nodes = a->n_nodes;
  p.n_q = a->n_q_heads;
  p.group = a->n_q_heads / a->n_kv_heads;
  p.rows = lay.rows;
  p.n_qt = lay.n_qt;
  p.n_pairs = lay.n_pairs;
  p.n_splits = lay.n_splits;
  p.row_pitch = lay.row_pitch;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  auto st = static_cast<cudaStream_t>(stream);
  return a->dtype == CBK_BF16 ? dispatch_tree<CBK_BF16>(a, p, st) : dispatch_tree<CBK_F16>(a, p, st);
}

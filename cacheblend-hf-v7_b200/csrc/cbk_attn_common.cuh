// Pieces of the attention kernels that feed tcgen05 (partial_attn_kernel,
// tree_attn_kernel): bounded waits that give way to an abort flag, the softmax
// arithmetic of a row in registers, and the K / V tensor maps.
#pragma once

#include <cuda.h>

#include "cbk_common.cuh"

namespace cbk {

constexpr int kBM = 128;       // rows per Q tile
constexpr int kBN = 128;       // keys per KV tile

// host side, cbk_attn.cu: SMs of the current device; 3-D map over [d2][d1][d0]
// 16-bit elements with row (d2) stride in elements, box {64, b1, b2}, 128-byte swizzle
int attn_sm_count();
int attn_make_map(CUtensorMap* m, const void* ptr, int dtype, uint64_t d0, uint64_t d1, uint64_t d2,
                  uint64_t row_stride, uint32_t b1, uint32_t b2);

__device__ __forceinline__ bool wait_or_abort(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  while (true) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (global_timer_ns() - t0 > kWaitLimitNs) return false;
  }
}

// two fp32 -> one packed 16-bit pair (lo in the low half), one conversion instruction
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (DT == CBK_BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// 32 fp32 values of a row times inv, rounded to the 16-bit type, stored to dst: as
// two 32-byte stores (whole sectors) when the caller's buffers are 32-byte aligned,
// else as four 16-byte stores.  The epilogue's stores are scattered rows (one row
// per thread), so whole-sector stores halve the requests and leave no partial sector.
template <int DT>
__device__ __forceinline__ void store_chunk(uint16_t* dst, const uint32_t (&o)[32], float inv, bool v8) {
  uint32_t w[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) w[e] = pack2<DT>(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
  if (v8) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                   :: "l"(dst + 16 * h), "r"(w[8 * h]), "r"(w[8 * h + 1]), "r"(w[8 * h + 2]), "r"(w[8 * h + 3]),
                      "r"(w[8 * h + 4]), "r"(w[8 * h + 5]), "r"(w[8 * h + 6]), "r"(w[8 * h + 7])
                   : "memory");
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) st_vec(dst + 8 * q, make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]));
  }
}

// max of three (one instruction on sm_100)
__device__ __forceinline__ float max3f(float a, float b, float c) {
  float m;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}

// (d0, d1) = (a0, a1) * (b, b) + (c, c) as one packed fp32 pair instruction
__device__ __forceinline__ void fma2(float& d0, float& d1, float a0, float a1, float b, float c) {
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %4};\n\tmov.b64 rc, {%5, %5};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d0), "=f"(d1) : "f"(a0), "f"(a1), "f"(b), "f"(c));
}

// (d0, d1) += (a0, a1) as one packed fp32 pair instruction
__device__ __forceinline__ void add2(float& d0, float& d1, float a0, float a1) {
  asm("{\n\t.reg .b64 ra, rd;\n\t"
      "mov.b64 rd, {%0, %1};\n\tmov.b64 ra, {%2, %3};\n\t"
      "add.f32x2 rd, rd, ra;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "+f"(d0), "+f"(d1) : "f"(a0), "f"(a1));
}

// packed fp32 pairs (two floats in one 64-bit register pair) for the f32x2 instructions
__device__ __forceinline__ uint64_t pk_f2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void upk_f2(uint64_t r, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul_f2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t sub_f2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// 2^x for a pair on the FMA pipe, to take load off the exponential unit.
// Split x = j + f with j = rint(x) (adding 1.5 * 2^23 leaves rint(x) in the low
// mantissa bits) and f in [-0.5, 0.5]; 2^f by a degree-3 polynomial, the
// minimax fit for relative error on [-0.5, 0.5] found with the Remez exchange
// algorithm (max relative error 7.5e-5, below the 16-bit rounding of P); 2^j is
// added into the exponent field.  x is clamped at -126 (j >= -126 keeps the
// exponent field from borrowing into the sign); below that the result is a
// denormal ~1e-38 instead of 0.
__device__ __forceinline__ void exp2_fma_pair(float x0, float x1, float& y0, float& y1) {
  constexpr float kMagic = 12582912.f;   // 1.5 * 2^23
  const uint64_t X = pk_f2(fmaxf(x0, -126.f), fmaxf(x1, -126.f));
  const uint64_t M = pk_f2(kMagic, kMagic);
  const uint64_t T = add_f2(X, M);
  const uint64_t F = sub_f2(X, sub_f2(T, M));
  uint64_t P = fma_f2(F, pk_f2(0.0551716685295105f, 0.0551716685295105f),
                      pk_f2(0.2426111251115799f, 0.2426111251115799f));
  P = fma_f2(P, F, pk_f2(0.6932609677314758f, 0.6932609677314758f));
  P = fma_f2(P, F, pk_f2(0.9999280571937561f, 0.9999280571937561f));
  float p0, p1, t0, t1;
  upk_f2(P, p0, p1);
  upk_f2(T, t0, t1);
  y0 = __int_as_float(__float_as_int(p0) + (__float_as_int(t0) << 23));
  y1 = __int_as_float(__float_as_int(p1) + (__float_as_int(t1) << 23));
}

// Pairs e (of the 16 per 32 columns; 3 of 16, the best of a 12-50 % sweep with PV
// split in halves and diagonal tiles masked in place; 6 of 16 was best before
// those) whose exponentials go to the FMA pipe; the others use ex2.approx.
#ifndef CBK_ATTN_EMU_MASK
#define CBK_ATTN_EMU_MASK 0x0421
#endif

// P = 2^(s * sl2 - m) of columns [32 c4, 32 c4 + 32) of a row, packed into 16-bit
// pairs, with the row sum accumulated in packed fp32 pairs.  3 of the 16 pairs go
// to the FMA-pipe polynomial (which drops a NaN argument).  Invisible keys arrive as s = -inf: ex2.approx gives
// 0 for them, the polynomial (its argument clamped at -126) 2^-126; with EMU = 0
// every pair takes ex2.approx, their weight is 0 exactly and NaN stays NaN.
template <int DT, unsigned EMU = CBK_ATTN_EMU_MASK>
__device__ __forceinline__ void exp_chunk(const uint32_t (&s)[kBN], int c4, float sl2, float neg_m,
                                          float& ra0, float& ra1, float& rb0, float& rb1, uint32_t (&pk)[16]) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int c = c4 * 32 + 2 * e;
    float x0, x1, p0, p1;
    fma2(x0, x1, __uint_as_float(s[c]), __uint_as_float(s[c + 1]), sl2, neg_m);
    if ((EMU >> e) & 1) {
      exp2_fma_pair(x0, x1, p0, p1);
    } else {
      p0 = ex2(x0);
      p1 = ex2(x1);
    }
    if (e & 1) add2(rb0, rb1, p0, p1);
    else add2(ra0, ra1, p0, p1);
    pk[e] = pack2<DT>(p0, p1);
  }
}

}  // namespace cbk

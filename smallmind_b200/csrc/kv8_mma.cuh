// Integer tensor-core pieces of the 8-bit KV cache's attention (mma.sync m16n8k32).
//
// The codes are the A operand as they are.  The fp32 side (q, or the softmax weights) enters as
// fixed point: three bytes of an integer of up to 23 bits, one MMA per byte, whose exact int32
// sums are put together in fp32.  No code is converted.  A value is off by half a step of 2^-22 (q, relative to its
// head's largest) or 2^-23 (weights times V scales, to the largest of a warp's keys) at most, where fp32's half step
// is 2^-24 of the value itself: far below what 8 bits of K and V cost, and a fourth digit would be a third more MMAs.
#pragma once
#include <cstdint>

#include "common.cuh"
#include "mma_i8.cuh"

namespace sm {

// D += A B, A s8 codes [16 x 32], B the 8-bit digits of 8 columns [32 x 8]
__device__ __forceinline__ void mma_s8u8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_u8s8_acc(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Bytes 0, 1 and 2 of four integers, each gathered into a word (integer 0 in the low byte).
__device__ __forceinline__ void bytes3(uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3, uint32_t& lo, uint32_t& mid,
                                       uint32_t& hi) {
  const uint32_t a = __byte_perm(x0, x1, 0x5140), b = __byte_perm(x2, x3, 0x5140);
  lo = __byte_perm(a, b, 0x5410);
  mid = __byte_perm(a, b, 0x7632);
  hi = __byte_perm(__byte_perm(x0, x1, 0x0062), __byte_perm(x2, x3, 0x0062), 0x5410);
}

// 4 x 4 bytes: w[i] holds columns 0..3 of row i; afterwards w[c] holds rows 0..3 of column c.
__device__ __forceinline__ void transpose4(uint32_t& w0, uint32_t& w1, uint32_t& w2, uint32_t& w3) {
  const uint32_t a = __byte_perm(w0, w1, 0x5140), b = __byte_perm(w2, w3, 0x5140);
  const uint32_t c = __byte_perm(w0, w1, 0x7362), d = __byte_perm(w2, w3, 0x7362);
  w0 = __byte_perm(a, b, 0x5410);
  w1 = __byte_perm(a, b, 0x7632);
  w2 = __byte_perm(c, d, 0x5410);
  w3 = __byte_perm(c, d, 0x7632);
}

// hi * 2^16 + mid * 2^8 + lo of three digit sums; join3_query: of a query's, |mid| and |lo| < 2^22, times 2^-22
__device__ __forceinline__ float join3_query(int hi, int mid, int lo) {
  return fmaf((float)hi, 0x1p-6f, (float)(mid * 256 + lo) * 0x1p-22f);
}
__device__ __forceinline__ float join3(int hi, int mid, int lo) {
  return fmaf((float)hi, 65536.f, fmaf((float)mid, 256.f, (float)lo));
}

// A query row's values are taken relative to 2^e, |x| < 2^e.  e stays at or above -120, where 2^e / sqrt(head_dim) is
// still a normal number: below it they lose bits, of 2^-143 and less.
__device__ __forceinline__ int query_exp(float peak) {
  return peak > 0.f ? max(((__float_as_int(peak) >> 23) & 0xFF) - 126, -120) : 0;
}
// x * 2^n in two steps, as 2^n itself may not be a normal number
struct Scale2 {
  float a, b;
  __device__ __forceinline__ explicit Scale2(int n) : a(pow2i(n / 2)), b(pow2i(n - n / 2)) {}
  __device__ __forceinline__ float operator()(float x) const { return x * a * b; }
};
// 2^e / sqrt(HD)
template <int HD>
__device__ __forceinline__ float query_unit(int e) {
  return pow2i(e - 1) * (HD == 64 ? 0.25f : 0.176776695f);
}

// Larger of the two, NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The softmax weight of x = score - maximum: (12 + 6x + x^2) / (12 - 6x + x^2) at max(x, -87.3).
// The reciprocal is the hardware's (1 ulp); a NaN stays one.
__device__ __forceinline__ float kv8_weight(float x) {
  const float c = max_nan(x, -87.3f);
  const float a = fmaf(c, c, 12.f);
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(-6.f, c, a)));
  return fmaf(6.f, c, a) * r;
}

// Two floats in one register pair, and their arithmetic in one instruction
struct Pair {
  uint64_t v;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ explicit Pair(float a) : Pair(a, a) {}
  __device__ __forceinline__ void get(float& a, float& b) const {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
  }
};
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// kv8_weight of two values
__device__ __forceinline__ Pair kv8_weight2(Pair x) {
  float a, b;
  x.get(a, b);
  const Pair c(max_nan(a, -87.3f), max_nan(b, -87.3f));
  const Pair s = fma2(c, c, Pair(12.f));
  fma2(c, Pair(-6.f), s).get(a, b);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(b));
  return mul2(fma2(c, Pair(6.f), s), Pair(a, b));
}

// Asynchronous copies into shared memory, in groups that a warp waits for itself
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// the same under an L2 policy
__device__ __forceinline__ uint64_t l2_evict_normal_policy() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy)
               : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {  // all but the N newest groups are here, for every lane
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
  __syncwarp();
}

}  // namespace sm

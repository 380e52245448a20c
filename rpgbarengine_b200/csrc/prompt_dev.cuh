// prompt_dev.cuh -- what the attention kernels on tcgen05 share (packed prompts, shared
// prefixes): paired fp32 operations, exponentials on the FMA pipe, operands from
// TMEM, TMEM loads that run beside other work.
#pragma once

#include <cuda_runtime.h>

#include "common.cuh"
#include "paged_dev.cuh"
#include "tc_dev.cuh"

namespace rpgc {
namespace paged {

// 32 bytes, a whole sector, at a 32-byte boundary.
RPGC_DEV void st_32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// Two fp32 operations at once.
RPGC_DEV uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
RPGC_DEV float2 unpair(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
RPGC_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
RPGC_DEV uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
RPGC_DEV uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 2^y of two values on the FMA pipe, for part of a row's probabilities: the
// special-function unit gives 16 exponentials per clock and SM, which takes as many clocks
// as the MMAs of the same tile with heads of 128 and twice as many with heads of 64.
// (One in eight: a quarter made 8192 tokens of heads of 128 slower; at 64 other shares
// have not been measured.)  y = n + f with n the nearest integer (added
// to and taken off 1.5 * 2^23 + 127), 2^f on [-1/2, 1/2] by a polynomial fitted to it
// for the smallest relative error (7.5e-5 for degree 3, 2.7e-6 for degree 4,
// against 2^-9 and 2^-12 of the 16-bit rounding that follows), times 2^n: the sum's
// last bits are n + 127, moved up they are the bits of 2^n.  For n = -127, where y
// stops, those of 0: -inf, the score of a key that the row does not see, has to give
// a weight of 0 (2^-126, which bf16 holds, times a value near its largest is 4).
// NaN is not carried (see `m`).
template <bool BF>
RPGC_DEV float2 exp2_poly(uint64_t y) {
  constexpr float kMagic = 12582912.0f + 127.0f;
  const float2 v = unpair(y);
  const uint64_t x = pair(fminf(max_nan(v.x, -127.0f), 127.0f), fminf(max_nan(v.y, -127.0f), 127.0f));
  const uint64_t t = add2(x, pair(kMagic, kMagic));
  const uint64_t f = fma2(add2(t, pair(-kMagic, -kMagic)), pair(-1.0f, -1.0f), x);
  uint64_t r;
  if (BF) {
    r = fma2(pair(0.0551716685f, 0.0551716685f), f, pair(0.242611125f, 0.242611125f));
    r = fma2(r, f, pair(0.693260968f, 0.693260968f));
    r = fma2(r, f, pair(0.999928057f, 0.999928057f));
  } else {
    r = fma2(pair(0.00957010221f, 0.00957010221f), f, pair(0.0559178591f, 0.0559178591f));
    r = fma2(r, f, pair(0.240247443f, 0.240247443f));
    r = fma2(r, f, pair(0.693121791f, 0.693121791f));
    r = fma2(r, f, pair(0.999999285f, 0.999999285f));
  }
  const float2 a = unpair(t);
  return unpair(mul2(r, pair(__uint_as_float(__float_as_uint(a.x) << 23), __uint_as_float(__float_as_uint(a.y) << 23))));
}
// V as the B operand of O += P V: rows are keys (the MMA's K), the 64 values
// of a panel row are N.  128-byte swizzle; 1024 B between groups of 8 keys,
// one panel between 64-column blocks.
RPGC_DEV uint64_t vdesc(const void* p, uint32_t panel) {
  const uint64_t a = smem_u32(p);
  return ((a >> 4) & 0x3FFFull) | ((uint64_t)(panel >> 4) << 16) | ((1024ull >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// True in one lane of a converged warp; the compiler knows that only one.
RPGC_DEV bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred P;\n elect.sync _|P, 0xffffffff;\n selp.b32 %0, 1, 0, P;\n}" : "=r"(p));
  return p != 0;
}

// D += A B with A (16-bit) in TMEM.
RPGC_DEV void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc));
}

// 32 consecutive columns of this warp's lanes; `r` holds them after tmem_landed.
RPGC_DEV void tmem_ld32_async(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// The registers pass through the wait, so that nothing uses them before it.
RPGC_DEV void tmem_landed(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
RPGC_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
RPGC_DEV void tmem_st16_nowait(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

}  // namespace paged
}  // namespace rpgc

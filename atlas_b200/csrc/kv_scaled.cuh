// Pieces shared by the kernels of the FP8 cache with a power of two per (page of 16 tokens, head): codes, scales, copies of pages, and which pages'
// softmax weights are not f16.
#pragma once
#include "common.cuh"

namespace atlas {

ATLAS_DEVICE int scale_exponent(float s) { return (int)((__float_as_uint(s) >> 23) & 255u) - 127; }
ATLAS_DEVICE float exact_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // e in [-126, 127]
ATLAS_DEVICE uint32_t e4m3x2_to_f16x2(uint32_t two) {                                            // the low half-word; exact
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(r) : "h"((uint16_t)two));
  return r;
}
ATLAS_DEVICE uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
ATLAS_DEVICE void bulk_page(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Softmax weights of pages whose value scales lie far apart.
//
// A token joins an output with p_j = 2^(s_j + ev - M), ev its page's value exponent.  A page's exponent is that of its largest token, so s_j + ev
// says too much of the others: one token 2^20 times as loud as everything else, itself without weight, lifts its fifteen neighbours by 20, and a
// reference M that followed them would push the p of all other pages out of f16.  Pages whose exponent is more than kFarApart away from that of
// the first or of the last page of what is attended over are therefore `far`: their p goes to the tensor cores as two bf16 terms (17 bits at any
// size; e4m3 is exact in bf16), and they move M only where they pass it by kFarSlack more than others.  The other pages' exponents are within
// 2 * kFarApart of each other, and their p has f16's 11 bits down to 2^-21 of what set M, steps of 2^-31 of it below: M stays kHeadroom below what
// set it, and moves when a score passes that by 2^8, so that p is below 2^15.  No limit of f16's or fp32's is met: far p below 2^47, sums of
// p 2^-ev below 2^107 a token.  (p itself ends at 2^-126: pages more than 100 powers quieter than others lose small weights.)  What is not told apart
// is loud and quiet tokens of one page: where every page has tokens 2^20 times as loud as those that carry the weight, loud tokens with weights
// below 2^-31 of the largest are lost.  e4m3 has lost the quiet ones' values by then: it ends 2^18 below a page's largest.  Exponents of trained
// caches lie within a few powers, and a far page costs a second product: were all pages far, 8 x 1024 prompt rows of 32 heads of 128 would take 147 us
// in place of 116, 517 rows of 16 heads of 256 behind 4096 tokens 70 in place of 57, 128 x 1152 single tokens 64 in place of 57.  Where none is,
// telling costs prompt rows 2 % (114 in place of 112 us, 56 of 55) and single tokens nothing.
constexpr int kFarApart = 8;
constexpr float kFarSlack = 32.f, kHeadroom = 7.f, kMoves = 15.f;
ATLAS_DEVICE bool exponents_apart(int a, int b) { return abs(a - b) > kFarApart; }
// the two bf16 terms of a pair of fp32 numbers
ATLAS_DEVICE void two_terms(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16x2(a, b);
  lo = pack_bf16x2(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xffff0000u));
}
ATLAS_DEVICE uint32_t h2_to_bf2(uint32_t v) {      // e4m3 numbers: exact in both
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
  return pack_bf16x2(f.x, f.y);
}

}  // namespace atlas

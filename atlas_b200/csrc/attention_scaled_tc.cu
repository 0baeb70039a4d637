// Chunk attention over the FP8 cache with a power-of-two scale per (page, head), on the 5th-generation tensor cores, and the softmax weight
// that each cached token got from a chunk's rows.
//
// As in attention_scaled.cu the codes are the operands and the scales live in the exponent: s_j = f q . k^_j with f = softmax scale * log2(e) * key
// page's scale, p_j = 2^(s_j + ev - M) in f16 or, in key tiles with a far page (kv_scaled.cuh), as two bf16 terms, o = sum p_j v^_j / sum p_j 2^-ev.
// A page covers 16 score columns, so f and ev - M are constants of a multiply-add over them, and a page's largest score is found before they are
// applied.
//
// scaled_chunk2_kernel (heads of 64 and 128), scaled_chunk_wide_kernel (256): tiles of 128 query rows of a key head; the G query heads of a key
// head are packed into the rows (row = token * G + head), so that a page is fetched and widened once for all of them.  One warp fetches pages
// (cp.async.bulk) and scales, others widen e4m3 to 16 bits into the 128-byte-swizzled K-major layout (values are stored with tokens along rows
// already), softmax takes a thread a row, and P goes back to TMEM over its scores as the operand of the next product.
//
// scaled_chunk_weigh_kernel: a cluster of two CTAs per (128 cached tokens, key head); tiles of the chunk's rows go by, every other one to each.
// S^T = K Q^T in bf16 (an e4m3 number is one exactly, and Q stays as it is): a TMEM lane is a token, so that the sum over rows and heads is a
// register's sum, and the two CTAs' sums are added in their order, with no atomics.
#include <type_traits>

#include "common.cuh"
#include "host_api.h"
#include "kv_scaled.cuh"
#include "tc_util.cuh"

namespace atlas {

constexpr int kScRows = 128;
constexpr int kScPg = 16;
constexpr int kScSub = 16 * 1024;                 // 128 rows x 64 16-bit numbers

struct ScChunkParams {
  const __nv_bfloat16* q; long long ldq; __nv_bfloat16* out; long long ldo;
  const uint8_t* k_cache; const uint8_t* v_cache;
  const float* k_scale; const float* v_scale; long long ks_ld, vs_ld; int ks_h, vs_h;
  const int* block_tables; int bt_ld, bt_cols;
  const int* seq_lens; const int* query_start_loc;
  const int* tile_seq; const int* tile_q0;
  float scale_log2;
  int Hq, Hkv, G, window, num_pages;
  float2* ml;                                     // [rows of the step][Hq] (M, 1 / l) or null
  // Few rows behind many keys: the keys of a query tile go to `splits` CTAs in equal shares, whose parts are joined by scaled_chunk_join_kernel
  int splits, first_row, rows;
  float* part_o; float2* part_ml;                 // [split][rows][Hq][D] and [split][rows][Hq] (M, l), rows from first_row on; no output of empty shares
  status_t* status;
};

ATLAS_DEVICE void sc_expect(uint64_t* bar, uint32_t bytes) {      // without arriving
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// The low word of a descriptor (make_smem_desc_sw128) carries the address, which steps along K; the high word is the same for all tiles.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
ATLAS_DEVICE uint32_t desc_low(const void* p) { return ((smem_u32(p) & 0x3FFFFu) >> 4) | (1u << 16); }
ATLAS_DEVICE void umma_f16_lo(uint32_t d_tmem, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 a, {%1, %5};\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
      : "memory");
}
ATLAS_DEVICE void sc_widen16(const uint4 v, uint4& lo, uint4& hi) {
  lo.x = e4m3x2_to_f16x2(v.x); lo.y = e4m3x2_to_f16x2(v.x >> 16); lo.z = e4m3x2_to_f16x2(v.y); lo.w = e4m3x2_to_f16x2(v.y >> 16);
  hi.x = e4m3x2_to_f16x2(v.z); hi.y = e4m3x2_to_f16x2(v.z >> 16); hi.z = e4m3x2_to_f16x2(v.w); hi.w = e4m3x2_to_f16x2(v.w >> 16);
}
ATLAS_DEVICE uint4 f16_to_bf16(uint4 v) { return make_uint4(h2_to_bf2(v.x), h2_to_bf2(v.y), h2_to_bf2(v.z), h2_to_bf2(v.w)); }

// A page whose table entry lies outside of the pool is skipped: its codes are zeros, which the copying warp puts where the copy would have gone,
// and its value exponent is -inf, so that no column of it has a weight.
ATLAS_DEVICE float2 skipped_page() { return make_float2(1.f, -INFINITY); }
template <int D>
ATLAS_DEVICE void clear_pages(uint8_t* stage, uint32_t pages) {      // the whole warp; 16 * D bytes a page
  const int lane = threadIdx.x & 31;
  for (uint32_t left = pages; left; left &= left - 1)
    for (int i = lane; i < D; i += 32) reinterpret_cast<uint4*>(stage)[(__ffs(left) - 1) * D + i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async();
  __syncwarp();
}

// Column of TMEM that holds channel `d` of the outputs (rows of the value tiles go there): of 32 channels 8 i + 2 k + e, column 8 k + 2 i + e.
// A load of 16 lanes x 256 bits gives thread 4 r + i columns 8 k + 2 i and one more of rows r and r + 8: eight channels in a row.
ATLAS_DEVICE int output_column(int d) { return (d & ~31) | (d & 6) << 2 | (d >> 2 & 6) | (d & 1); }
// Channel of 32 for a lane that widens values: eight neighbouring lanes have channels, and output columns, that differ modulo 8 (no two of them
// in the same banks, neither reading nor writing).
ATLAS_DEVICE int value_piece(int r) {
  const int i = r >> 1 & 3, k = (i + (r >> 3)) & 3;
  return (r & ~31) | 8 * i + 2 * k | (r & 1);
}
ATLAS_DEVICE void tmem_ld_16x256b_x8(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,"
      "%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// A warp's 32 rows of outputs, times 1 / l to bf16, or as they are to a part of the row.  at: where this lane's row begins, -1 where it is not
// stored; done() when TMEM has been read.  A store writes 64 bytes of eight rows (a row a lane, 16 bytes of 32 rows, took 4500 clocks for two
// tiles).
template <int D, typename Done>
ATLAS_DEVICE void store_outputs(uint32_t tO, bool zeros, float inv, long long at, __nv_bfloat16* out, float* part, Done done) {
  const int lane = threadIdx.x & 31, ch = (lane & 3) * 8;
#pragma unroll 1
  for (int g = 0; g < 2; ++g) {
    float f[2];
    long long to[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f[h] = __shfl_sync(0xffffffffu, inv, g * 16 + h * 8 + (lane >> 2));
      to[h] = __shfl_sync(0xffffffffu, at, g * 16 + h * 8 + (lane >> 2));
    }
#pragma unroll 1
    for (int c = 0; c < D; c += 64) {
      uint32_t r[32];
      if (zeros) {
#pragma unroll
        for (int i = 0; i < 32; ++i) r[i] = 0;
      } else {
        tmem_ld_16x256b_x8(tO + (g << 20) + c, r);
        tmem_ld_wait();
      }
      if (g == 1 && c + 64 == D) done();
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (to[h] < 0) continue;
          const uint32_t* v = r + 16 * u + 2 * h;
          if (part) {
            float* o = part + to[h] + c + 32 * u + ch;
            *reinterpret_cast<uint4*>(o) = make_uint4(v[0], v[1], v[4], v[5]);
            *reinterpret_cast<uint4*>(o + 4) = make_uint4(v[8], v[9], v[12], v[13]);
          } else {
            uint4 o;
            o.x = pack_bf16x2(__uint_as_float(v[0]) * f[h], __uint_as_float(v[1]) * f[h]);
            o.y = pack_bf16x2(__uint_as_float(v[4]) * f[h], __uint_as_float(v[5]) * f[h]);
            o.z = pack_bf16x2(__uint_as_float(v[8]) * f[h], __uint_as_float(v[9]) * f[h]);
            o.w = pack_bf16x2(__uint_as_float(v[12]) * f[h], __uint_as_float(v[13]) * f[h]);
            *reinterpret_cast<uint4*>(out + to[h] + c + 32 * u + ch) = o;
          }
        }
    }
  }
}

// The shares of a row: o = sum_s o_s 2^(M_s - M) / sum_s l_s 2^(M_s - M); a warp a (row, head).
template <int D>
__global__ void __launch_bounds__(256)
scaled_chunk_join_kernel(const ScChunkParams p) {
  const int lane = threadIdx.x & 31;
  const long long u = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const long long step = (long long)p.rows * p.Hq;
  if (u >= step) return;
  const long long row = p.first_row + u / p.Hq;
  const int head = (int)(u % p.Hq);
  float m = -INFINITY;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, p.part_ml[s * step + u].x);
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f, o[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) o[i] = 0.f;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float2 x = p.part_ml[s * step + u];
    const float f = fast_exp2(x.x - ref);
    l += x.y * f;
    if (x.x == -INFINITY) continue;                              // a share that the row sees nothing of may have no output
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const float2 y = *reinterpret_cast<const float2*>(p.part_o + (s * step + u) * D + i * 64 + lane * 2);
      o[2 * i] = fmaf(y.x, f, o[2 * i]);
      o[2 * i + 1] = fmaf(y.y, f, o[2 * i + 1]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < D / 64; ++i)
    *reinterpret_cast<uint32_t*>(p.out + row * p.ldo + head * D + i * 64 + lane * 2) = pack_bf16x2(o[2 * i] * inv, o[2 * i + 1] * inv);
  if (p.ml && lane == 0) p.ml[row * p.Hq + head] = make_float2(ref, inv);
}

// ---------------------------------------------------------------------------------------------------------------- two tiles at a time
// Heads of 64 and 128: two query tiles share every widened key tile.  Persistent, one CTA per SM; items (pair of query tiles, key head) with the
// most keys first.
//   warps 0..3, 4..7   softmax of tile A and of tile B, a thread a row
//   warps 8..11        keys to bf16, values to f16 (two buffers of each)
//   warps 12, 14       products of tile A and of tile B, by halves of a key tile: scores of 64 keys go behind the product that read P out of
//                      the same columns, so that the softmax finds the next half ready (whole key tiles: 138 in place of 115 us, 8 x 1024 rows)
//   warp 13            the items, and query tiles by TMA, as they are (bf16: keys are exact in it)
//   warp 15            pages by bulk copies, their scales
// Per pair of tiles and 128 keys: products 2048 clocks of the tensor cores, exponentials 2048 of the special-function units, shared memory 2048
// for operands, 512 for the widened tiles and 512 for the codes.  Measured 5000: a softmax thread's chain of 2500 for 64 keys, half of it
// exponentials shared by two warps a scheduler; no unit is busy for more than half of the time (issue slots 47 %, tensor cores 42 %, special
// functions 35 %: profiles/kv_scaled_cache.md).  Rounds of 16 or 32 columns, a part of the exponentials as polynomials, and the tiles half a step
// apart were slower or no faster.  8 x 1024 rows of 32 heads of 128: 114 us, 602 TFLOP/s; two sequences of 3001 rows: 152.
constexpr int kC2Threads = 512;
constexpr int kC2Kv = 128, kC2Pages = 8, kC2Ring = 8, kC2Scales = kC2Pages + 1;

template <int D>
struct C2Tile {
  static constexpr int kQ = (D / 64) * kScSub;                    // a query tile
  static constexpr int kK = (D / 64) * kScSub;                    // 128 keys
  static constexpr int kV = 2 * D * 128;                          // D channels x 128 tokens
  static constexpr int kStage = kC2Kv * D;                        // the pages of a key tile
  static constexpr int kSmem = 2 * (kQ + kK + kV) + 2 * kStage + kC2Ring * kC2Scales * 8 + 448 + 1024;      // at most 227 KB
};

// A from TMEM: a row a lane, two 16-bit numbers a column
ATLAS_DEVICE void umma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_low), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
      : "memory");
}
ATLAS_DEVICE void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// pairs of fp32 numbers in one instruction
ATLAS_DEVICE uint64_t pair2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
ATLAS_DEVICE float2 unpair2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
ATLAS_DEVICE uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
ATLAS_DEVICE uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

ATLAS_DEVICE uint32_t bits_below(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }
ATLAS_DEVICE float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// A row's step over 64 score columns (a thread a row): their largest s + ev, then p = 2^(s + ev - m) as f16 over the first half of the columns
// at tP, or, where the key tile has a far page (kv_scaled.cuh), as two bf16 terms over both halves.  f: (score factor, value exponent) of the four
// pages; columns [lo, hi) are visible.  The reference m moves only when a score passes what set it by 2^8 (p stays inside f16), which is rare
// after a row's first columns; the output, where there is one, then moves with it, after wait_output() has seen the last product that goes to
// it.  False: that wait ran out.
template <int D, bool kFar, typename Wait>
ATLAS_DEVICE bool softmax_step(uint32_t tS, uint32_t tP, uint32_t tO, const float2 (&f)[4], bool whole, int hi, int lo, bool output, float& m,
                               float& l, Wait wait_output) {
  uint32_t v[2][32];
  tmem_ld_32x32b_x32(tS, v[0]);
  tmem_ld_32x32b_x32(tS + 32, v[1]);
  tmem_ld_wait();
  if (!whole) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t seen = bits_below(hi - k * 32) & ~bits_below(lo - k * 32);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[k][i] = (seen >> i) & 1u ? v[k][i] : 0xff800000u;
    }
  }
  float mx[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t* u = &v[q >> 1][(q & 1) * 16];
    float a = __uint_as_float(u[0]), z = __uint_as_float(u[1]);
#pragma unroll
    for (int i = 2; i < 14; i += 4) {
      a = max3_nan(a, __uint_as_float(u[i]), __uint_as_float(u[i + 1]));
      z = max3_nan(z, __uint_as_float(u[i + 2]), __uint_as_float(u[i + 3]));
    }
    a = max3_nan(a, __uint_as_float(u[14]), __uint_as_float(u[15]));
    mx[q] = fmaf(max3_nan(a, z, z), f[q].x, f[q].y);
  }
  const float top = max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]) - (kFar ? kFarSlack : 0.f);
  if (__any_sync(0xffffffffu, !(top <= m + kMoves))) {            // NaN too: the row is NaN from here on
    float alpha = 1.f;
    if (!(top <= m + kMoves)) {
      alpha = (m == -INFINITY) ? 0.f : fast_exp2(m - (top - kHeadroom));
      m = top - kHeadroom;
    }
    l *= alpha;
    if (output) {
      if (!wait_output()) return false;
      tc_fence_after();
#pragma unroll 1
      for (int k = 0; k < D / 16; ++k) {
        uint32_t o[16];
        tmem_ld_32x32b_x16(tO + k * 16, o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
        tmem_st_32x32b_x16(tO + k * 16, o);
      }
    }
  }
  const float ref = (m == -INFINITY) ? 0.f : m;
  // p of page q, two columns at a time: put(column / 2, p, p)
  auto page = [&](int q, auto put) {
    const uint32_t* u = &v[q >> 1][(q & 1) * 16];
    const float add = f[q].y - ref;
    const uint64_t f2 = pair2(f[q].x, f[q].x), a2 = pair2(add, add);
    uint64_t s2 = 0;
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const uint64_t x2 = fma2(pair2(__uint_as_float(u[i]), __uint_as_float(u[i + 1])), f2, a2);
      float2 e = unpair2(x2);
      e.x = fast_exp2(e.x);
      e.y = fast_exp2(e.y);
      s2 = add2(s2, pair2(e.x, e.y));
      put(i / 2, e.x, e.y);
    }
    const float2 s = unpair2(s2);
    l = fmaf(s.x + s.y, exact_pow2((int)fminf(-f[q].y, 127.f)), l);      // a skipped page: 0 times anything
  };
  if constexpr (!kFar) {
    uint32_t w[2][16];
#pragma unroll
    for (int q = 0; q < 4; ++q) page(q, [&](int i, float a, float b) { w[q >> 1][(q & 1) * 8 + i] = pack_f16x2(a, b); });
    tmem_st_32x32b_x16(tP, w[0]);
    tmem_st_32x32b_x16(tP + 16, w[1]);
  } else {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t hi2[16], lo2[16];
#pragma unroll
      for (int q = 0; q < 2; ++q) page(2 * k + q, [&](int i, float a, float b) { two_terms(a, b, hi2[q * 8 + i], lo2[q * 8 + i]); });
      tmem_st_32x32b_x16(tP + 16 * k, hi2);
      tmem_st_32x32b_x16(tP + 32 + 16 * k, lo2);
    }
  }
  tmem_st_wait();
  return true;
}

// The value scales (powers of two) of pages that are not far: of the first page of the CTA's keys and the sequence's newest one, 0 where that is
// not in the pool.
struct NearScales {
  float least, most;
  ATLAS_DEVICE void begin(float first, float last) {
    if (first == 0.f) first = last;
    if (last == 0.f) last = first;
    least = fmaxf(first, last) * exact_pow2(-kFarApart);
    most = first == 0.f ? INFINITY : fminf(first, last) * exact_pow2(kFarApart);
  }
  ATLAS_DEVICE bool far(float scale) const { return scale < least || scale > most; }
};

struct alignas(16) C2Item {
  int b, kvh, split, L, q_row0, q_len, q0, ctx0, page0;           // b < 0: no more; page0: the first of this share of the keys
  int n[2], n_kv;                                                 // key tiles of tile A, of tile B, of both
};
// Item of a CTA in round `rd`: the rounds go to and fro over the CTAs, so that the ones with the longest item of a round get the shortest of
// the next (2 x 3001 ragged rows: 47 key tiles on the busiest CTA of 44 on average, 56 with rounds all one way).
ATLAS_DEVICE C2Item c2_item(const ScChunkParams& p, int rd, int items) {
  const int it = rd * (int)gridDim.x + ((rd & 1) ? (int)(gridDim.x - 1 - blockIdx.x) : (int)blockIdx.x);
  C2Item r;
  r.b = -1;
  if (it >= items) return r;
  const int tile = it / (p.Hkv * p.splits), toks = kScRows / p.G;
  r.b = p.tile_seq[tile];
  r.q0 = p.tile_q0[tile];
  r.kvh = it % p.Hkv;
  r.split = it / p.Hkv % p.splits;
  r.L = min(p.seq_lens[r.b], p.bt_cols * kScPg);
  r.q_row0 = p.query_start_loc[r.b];
  r.q_len = p.query_start_loc[r.b + 1] - r.q_row0;
  r.ctx0 = r.L - r.q_len;
  r.page0 = p.window > 0 ? max(r.ctx0 + r.q0 - p.window + 1, 0) / kScPg : 0;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int first = r.q0 + x * toks, last = min(first + toks, r.q_len);
    r.n[x] = first < r.q_len ? max((min(r.L, r.ctx0 + last) - r.page0 * kScPg + kC2Kv - 1) / kC2Kv, 0) : 0;
  }
  if (p.splits > 1) {
    const int share = (max(r.n[0], r.n[1]) + p.splits - 1) / p.splits;
    r.page0 += r.split * share * kC2Pages;
#pragma unroll
    for (int x = 0; x < 2; ++x) r.n[x] = min(max(r.n[x] - r.split * share, 0), share);
  }
  r.n_kv = max(r.n[0], r.n[1]);
  return r;
}

template <int D>
__global__ void __launch_bounds__(kC2Threads, 1)
scaled_chunk2_kernel(const __grid_constant__ CUtensorMap tmap_q, const ScChunkParams p, int items) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using Tile = C2Tile<D>;
  uint8_t* sQ = smem;                                             // tile A, tile B: D / 64 sub-tiles [128 rows][64 channels]
  uint8_t* sK = sQ + 2 * Tile::kQ;                                // two buffers: D / 64 sub-tiles [128 tokens][64 channels]
  uint8_t* sV = sK + 2 * Tile::kK;                                // two buffers: 2 sub-tiles [D channels][64 tokens]
  uint8_t* sStK = sV + 2 * Tile::kV;                              // the pages as they come, keys and values
  uint8_t* sStV = sStK + Tile::kStage;
  float2* sScale = reinterpret_cast<float2*>(sStV + Tile::kStage);  // [kC2Ring][8 pages: (score factor, value exponent); is one far?]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sScale + kC2Ring * kC2Scales);
  uint64_t* q_full = bars;
  uint64_t* q_free = bars + 1;                                    // the item's last QK
  uint64_t* k_full = bars + 2;                                    // [2] 4 warps
  uint64_t* k_free = bars + 4;                                    // [2] QK of both tiles
  uint64_t* v_full = bars + 6;                                    // [2] 4 warps
  uint64_t* v_free = bars + 8;                                    // [2] PV of both tiles
  uint64_t* s_full = bars + 10;                                   // [tile][half]
  uint64_t* p_ready = bars + 22;                                  // [tile][half] 4 warps
  uint64_t* pv_done = bars + 14;                                  // [tile]
  uint64_t* o_free = bars + 16;                                   // [tile] 4 warps have read the item's output
  uint64_t* ks_full = bars + 18;                                  // [keys, values] pages have come
  uint64_t* ks_free = bars + 20;                                  // [keys, values] 4 warps
  uint64_t* pv_half = bars + 26;                                  // [tile] the first half's product
  uint64_t* item_full = bars + 28;                                // [2] warp 13
  uint64_t* item_free = bars + 30;                                // [2] the 15 other warps have read it
  C2Item* sItem = reinterpret_cast<C2Item*>(bars + 32);           // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sItem + 2);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.G, toks = kScRows / G;

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) { mbar_init(&ks_full[s], 1); mbar_init(&ks_free[s], 4); }
    mbar_init(q_full, 1); mbar_init(q_free, 2);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], 4); mbar_init(&k_free[s], 2); mbar_init(&v_full[s], 4); mbar_init(&v_free[s], 2);
      mbar_init(&pv_done[s], 1); mbar_init(&pv_half[s], 1); mbar_init(&o_free[s], 4);
    }
    for (int s = 0; s < 4; ++s) { mbar_init(&s_full[s], 1); mbar_init(&p_ready[s], 4); }
    for (int s = 0; s < 2; ++s) { mbar_init(&item_full[s], 1); mbar_init(&item_free[s], 15); }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 12) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  if (warp == 13 && lane == 0) tma_prefetch_desc(&tmap_q);
  // rows behind a tile's last whole token are never loaded: zeros (whatever lay there could be NaN, which sends its warp through the rare path)
  for (int i = threadIdx.x; i < 2 * (D / 64) * (kScRows - toks * G) * 8; i += kC2Threads) {
    const int rest = kScRows - toks * G, row = toks * G + (i >> 3) % rest, sub = (i >> 3) / rest;
    *reinterpret_cast<uint4*>(sQ + sub * kScSub + row * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;                               // scores of A, of B (128 columns each, P over them), outputs of A, of B

  // Every role but warp 13 gets the CTA's items from shared memory.  (Each role working them out for itself, in a copy of that code of its own
  // that was cold by the next item, took 5000 clocks an item.)
  uint32_t n_item = 0;
  C2Item m_;
  auto next = [&]() -> bool {
    const uint32_t s = n_item & 1;
    const bool got = mbar_wait(&item_full[s], (n_item >> 1) & 1, abort_flag, p.status, 0xC40);
    if (!__all_sync(0xffffffffu, got)) return false;
    m_ = sItem[s];
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_free[s]);
    ++n_item;
    return m_.b >= 0;
  };

  if (warp < 8) {
    // ------------------------------------------------------------------ softmax: tile x, a thread a row
    const int x = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t t_lane = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + x * 128 + t_lane, tO = tmem + 256 + x * D + t_lane;
    int n_s = 0, ring = 0;                                        // score tiles of this tile so far, key tiles of both
    bool ok = true;
    while (ok && next()) {
      const int n = m_.n[x];
      const int tok = m_.q0 + x * toks + row / G, head = m_.kvh * G + row % G;
      const bool live = row < toks * G && tok < m_.q_len;
      const int pos = m_.ctx0 + tok;
      // keys [start, end) are visible; rows that are not there see all, so that their warp need not mask, and are not stored
      const int end = live ? min(pos + 1, m_.L) : 1 << 30;
      const int start = live && p.window > 0 ? pos - p.window + 1 : 0;
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < n; ++j) {
        ++n_s;
        const int kv0 = (m_.page0 + j * kC2Pages) * kScPg;
        const int hi = end - kv0, lo = start - kv0;
        const bool whole = __all_sync(0xffffffffu, hi >= kC2Kv && lo <= 0);
        const float2* sc = sScale + ((ring + j) % kC2Ring) * kC2Scales;
        // ---- 64 columns at a time; P takes half of the columns that its scores had
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {                               // no further unrolled: the roles' code shares one instruction cache
          ok = mbar_wait(&s_full[2 * x + c], (n_s - 1) & 1, abort_flag, p.status, 0xC00 + x);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          tc_fence_after();
          float2 f[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) f[q] = sc[c * 4 + q];
          auto output_there = [&] {
            return (bool)__all_sync(0xffffffffu, mbar_wait(c ? &pv_half[x] : &pv_done[x], (n_s - 2 + c) & 1, abort_flag, p.status, 0xC04 + x));
          };
          ok = sc[kC2Pages].x == 0.f
                   ? softmax_step<D, false>(tS + c * 64, tS + c * 64, tO, f, whole, hi - c * 64, lo - c * 64, j > 0 || c == 1, m, l, output_there)
                   : softmax_step<D, true>(tS + c * 64, tS + c * 64, tO, f, whole, hi - c * 64, lo - c * 64, j > 0 || c == 1, m, l, output_there);
          if (!ok) break;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_ready[2 * x + c]);          // the first half's product runs under the second half
        }
        if (!ok) break;
      }
      ring += m_.n_kv;
      if (!ok) break;
      // ---- o / l, or this share's o and l
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const long long at = (long long)(m_.q_row0 + tok) * p.Hq + head, at_part = ((long long)m_.split * p.rows - p.first_row) * p.Hq + at;
      const bool part = p.splits > 1;
      if (n > 0) {
        ok = mbar_wait(&pv_done[x], (n_s - 1) & 1, abort_flag, p.status, 0xC02 + x);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc_fence_after();
      }
      store_outputs<D>(tO, n == 0, inv, !live || (part && n == 0) ? -1 : part ? at_part * D : (long long)(m_.q_row0 + tok) * p.ldo + head * D, p.out, part ? p.part_o : nullptr, [&] {
        if (n == 0) return;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[x]);
      });
      if (live) {
        if (part) p.part_ml[at_part] = make_float2(m, l);
        else if (p.ml) p.ml[at] = make_float2(m == -INFINITY ? 0.f : m, inv);
      }
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------------ converters
    const int r = threadIdx.x - 256;
    constexpr int kPer = D / 16;                                  // 16-byte pieces of a thread and tile: piece i of page i / D
    uint32_t n_t = 0;                                             // key tiles so far
    bool ok = true;
    while (ok && next()) {
      const int L = m_.L, page0 = m_.page0, n_kv = m_.n_kv;
      for (int j = 0; j < n_kv; ++j, ++n_t) {
        const int s = n_t & 1;
        // ---- keys
        ok = mbar_wait(&ks_full[0], n_t & 1, abort_flag, p.status, 0xC10) &&
             mbar_wait(&k_free[s], ((n_t >> 1) & 1) ^ 1u, abort_flag, p.status, 0xC11);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
#pragma unroll 4
        for (int k = 0; k < kPer; ++k) {
          // eight neighbouring lanes take 64 bytes each of two rows, with heads of 128 from different sub-tiles: no two of their loads or
          // stores fall into the same banks
          const int i = k * 128 + r, trow = D == 128 ? k * kScPg + (r >> 5) * 4 + (r >> 4 & 1) * 2 + ((r >> 2 ^ r >> 3) & 1) : i / 4;
          const int c = D == 128 ? r & 7 : i % 4, tsw = trow & 7;
          uint4 lo, hi;
          sc_widen16(reinterpret_cast<const uint4*>(sStK)[trow * (D / 16) + c], lo, hi);
          uint8_t* rowp = sK + s * Tile::kK + (c >> 2) * kScSub + (trow >> 3) * 1024 + tsw * 128;
          const int ch = (c & 3) * 2;
          *reinterpret_cast<uint4*>(rowp + ((ch ^ tsw) << 4)) = f16_to_bf16(lo);
          *reinterpret_cast<uint4*>(rowp + (((ch + 1) ^ tsw) << 4)) = f16_to_bf16(hi);
        }
        fence_proxy_async();                                      // the tile for the products, and the pages read before they are copied over
        __syncwarp();
        if (lane == 0) { mbar_arrive(&k_full[s]); mbar_arrive(&ks_free[0]); }
        // ---- values
        ok = mbar_wait(&ks_full[1], n_t & 1, abort_flag, p.status, 0xC12) &&
             mbar_wait(&v_free[s], ((n_t >> 1) & 1) ^ 1u, abort_flag, p.status, 0xC13);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        auto widen = [&](auto far) {                              // a far page: bf16; the usual loop stays free of that
#pragma unroll 4
          for (int k = 0; k < kPer; ++k) {
            const int i = k * 128 + value_piece(r), pg = i / D, dim = i % D, col = output_column(dim), sw = col & 7;
            const int left = L - (page0 + j * kC2Pages + pg) * kScPg;      // tokens of the page; the others are cleared
            uint4 v = reinterpret_cast<const uint4*>(sStV)[i];
            if (left < kScPg) {
              uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const int there = min(max(left - 4 * q, 0), 4);
                w[q] = there == 4 ? w[q] : (w[q] & ((1u << (8 * there)) - 1u));
              }
            }
            uint4 lo, hi;
            sc_widen16(v, lo, hi);
            if constexpr (decltype(far)::value) { lo = f16_to_bf16(lo); hi = f16_to_bf16(hi); }
            uint8_t* rowp = sV + s * Tile::kV + (pg >> 2) * (D * 128) + col * 128;
            const int ch = (pg & 3) * 2;
            *reinterpret_cast<uint4*>(rowp + ((ch ^ sw) << 4)) = lo;
            *reinterpret_cast<uint4*>(rowp + (((ch + 1) ^ sw) << 4)) = hi;
          }
        };
        if (sScale[n_t % kC2Ring * kC2Scales + kC2Pages].x == 0.f) widen(std::false_type{});
        else widen(std::true_type{});
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) { mbar_arrive(&v_full[s]); mbar_arrive(&ks_free[1]); }
      }
    }
  } else if (warp == 15) {
    // ------------------------------------------------------------------ pages: lanes 0..7 keys, 8..15 values, entries and scales two tiles ahead
    const bool is_v = (lane & 8) != 0;
    uint32_t n_t = 0;
    bool ok = true;
    while (ok && next()) {
      const int n_pages = (m_.L + kScPg - 1) / kScPg;
      const int* bt = p.block_tables + (long long)m_.b * p.bt_ld;
      auto entry = [&](int j) {                                   // -1: behind the end or outside of the pool
        const int pg = m_.page0 + j * kC2Pages + (lane & 7);
        return lane < 16 && j < m_.n_kv && pg < n_pages ? bt[pg] : -1;
      };
      auto scale_of = [&](int blk) {
        if ((unsigned)blk >= (unsigned)p.num_pages) return 1.f;
        return is_v ? p.v_scale[blk * p.vs_ld + m_.kvh * p.vs_h] : p.k_scale[blk * p.ks_ld + m_.kvh * p.ks_h];
      };
      const int newest = n_pages > 0 ? bt[n_pages - 1] : -1;
      int blk = entry(0), blk1 = entry(1);
      const float last = (unsigned)newest < (unsigned)p.num_pages ? p.v_scale[newest * p.vs_ld + m_.kvh * p.vs_h] : 0.f;
      float sc = scale_of(blk);
      NearScales near;
      for (int j = 0; j < m_.n_kv; ++j, ++n_t) {
        const int blk2 = entry(j + 2);
        const float sc1 = scale_of(blk1);
        const bool live = (unsigned)blk < (unsigned)p.num_pages;
        const uint32_t pages = __ballot_sync(0xffffffffu, live);
        const bool skip = lane < 8 && m_.page0 + j * kC2Pages + lane < n_pages && !live;
        const uint32_t skipped = __ballot_sync(0xffffffffu, skip);
        const long long at = ((long long)blk * p.Hkv + m_.kvh) * (kScPg * D);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          ok = mbar_wait(&ks_free[w], (n_t & 1) ^ 1u, abort_flag, p.status, 0xC30 + w);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          if (skipped) clear_pages<D>(w ? sStV : sStK, skipped);
          if (lane == 0) sc_expect(&ks_full[w], (uint32_t)__popc((pages >> (8 * w)) & 0xFFu) * (kScPg * D));
          __syncwarp();
          if (live && is_v == (w == 1)) bulk_page((w ? sStV : sStK) + (lane & 7) * (kScPg * D), (w ? p.v_cache : p.k_cache) + at, kScPg * D, &ks_full[w]);
          if (w == 0) {                                             // under the copies: the scales may not be there yet
            const float vs = __shfl_sync(0xffffffffu, sc, 8 + (lane & 7));
            if (j == 0) near.begin(pages >> 8 & 1 ? __shfl_sync(0xffffffffu, sc, 8) : 0.f, last);
            const bool far = __any_sync(0xffffffffu, live && is_v && near.far(sc));
            float2* to = sScale + n_t % kC2Ring * kC2Scales;
            if (lane < 8) to[lane] = skip ? skipped_page() : make_float2(p.scale_log2 * sc, (float)scale_exponent(vs));
            if (lane == 8) to[kC2Pages].x = far;
            __syncwarp();
          }
          if (lane == 0) mbar_arrive(&ks_full[w]);
        }
        if (!ok) break;
        blk = blk1; blk1 = blk2;
        sc = sc1;
      }
    }
    if (*abort_flag)
      for (int i = 0; i < 64; ++i) __nanosleep(1000);
  } else if (warp == 12 || warp == 14) {
    // ------------------------------------------------------------------ products of tile x, each tile at its own pace.  The whole warp walks the
    // list and one elected lane issues: descriptors stay in uniform registers so (under a lane's branch an MMA took 110 clocks to issue).
    constexpr uint32_t kIdescS = make_idesc(kScRows, 64, 1u);      // bf16 scores
    constexpr uint32_t kIdescO = make_idesc(kScRows, D, 0u), kIdescFar = make_idesc(kScRows, D, 1u);      // f16 outputs; bf16, of two terms
    const int x = (warp - 12) >> 1;
    const uint32_t dQ = desc_low(sQ + x * Tile::kQ), dK = desc_low(sK), dV = desc_low(sV);
    const uint32_t tS = tmem + x * 128, tO = tmem + 256 + x * D;
    uint32_t n_t = 0, n_i = 0, pvs = 0, outs = 0;   // key tiles, items, PV products, items with output
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t site) { return (bool)__all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.status, site + x)); };
    auto full = [&](uint64_t* bar, uint32_t t, uint32_t site) { return wait(bar + (t & 1), (t >> 1) & 1, site); };
    // scores with half of key tile t; the PV product that read P out of the same columns is done
    auto score = [&](uint32_t t, int half, bool last) -> bool {
      if (pvs > 0 && !wait(half ? &pv_done[x] : &pv_half[x], (pvs - 1) & 1, 0xC20)) return false;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t bd = dK + (t & 1) * (Tile::kK >> 4) + half * (64 * 128 >> 4);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t at = (ks >> 2) * (kScSub >> 4) + 2 * (ks & 3);
          umma_f16_lo(tS + half * 64, dQ + at, bd + at, kIdescS, ks > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[2 * x + half]);
        if (half) {
          umma_commit(&k_free[t & 1]);
          if (last) umma_commit(q_free);
        }
      }
      __syncwarp();
      return true;
    };
    // a tile that has no use for a buffer hands it on, once it is full (its last use is counted then)
    auto skip = [&](uint64_t* bar_free, uint32_t t) {
      if (lane == 0) mbar_arrive(bar_free + (t & 1));
    };
    for (; ok && next(); ++n_i) {
      const int n = __shfl_sync(0xffffffffu, m_.n[x], 0), n_kv = __shfl_sync(0xffffffffu, m_.n_kv, 0);
      ok = wait(q_full, n_i & 1, 0xC22);
      if (!ok) break;
      if (n == 0 && lane == 0) mbar_arrive(q_free);
      if (n_kv == 0) continue;
      ok = full(k_full, n_t, 0xC24);
      if (ok && n > 0) ok = score(n_t, 0, false) && score(n_t, 1, n == 1);
      else if (ok) skip(k_free, n_t);
      for (int j = 0; j < n_kv && ok; ++j, ++n_t) {
        // what the next products need besides P, before P is waited for
        ok = full(v_full, n_t, 0xC26) && (j + 1 >= n_kv || full(k_full, n_t + 1, 0xC2C));
        if (!ok) break;
        if (j < n) {
          if (j == 0 && outs > 0) ok = wait(&o_free[x], (outs - 1) & 1, 0xC28);
          for (int half = 0; half < 2 && ok; ++half) {
            ok = wait(&p_ready[2 * x + half], (pvs - half) & 1, 0xC2A);
            if (!ok) break;
            tc_fence_after();
            const bool far = sScale[n_t % kC2Ring * kC2Scales + kC2Pages].x != 0.f;
            if (elect_one()) {
              const uint32_t tP = tS + half * 64, bd = dV + (n_t & 1) * (Tile::kV >> 4) + half * (D * 128 >> 4);
              const uint32_t more = j > 0 || half > 0;
              if (!far) {
#pragma unroll
                for (int ks = 0; ks < kC2Kv / 32; ++ks) umma_f16_ta(tO, tP + ks * 8, bd + 2 * ks, kIdescO, ks > 0 ? 1u : more);
              } else {
#pragma unroll
                for (int ks = 0; ks < kC2Kv / 16; ++ks) umma_f16_ta(tO, tP + ks * 8, bd + 2 * (ks % 4), kIdescFar, ks > 0 ? 1u : more);
              }
              if (half == 0) {
                umma_commit(&pv_half[x]);
              } else {
                umma_commit(&pv_done[x]);
                umma_commit(&v_free[n_t & 1]);
              }
            }
            __syncwarp();
            if (half == 0) ++pvs;
            if (j + 1 < n) ok = score(n_t + 1, half, j + 2 == n);
          }
          if (!ok) break;
          if (j + 1 == n) ++outs;
        } else {
          skip(v_free, n_t);
        }
        if (j + 1 < n_kv && j + 1 >= n) skip(k_free, n_t + 1);
      }
    }
  } else if (warp == 13) {
    // ------------------------------------------------------------------ items, two ahead, and their query tiles
    if (lane == 0) {
      bool ok = true;
      auto publish = [&](int rd) {
        ok = mbar_wait(&item_free[rd & 1], ((rd >> 1) & 1) ^ 1u, abort_flag, p.status, 0xC31);
        if (!ok) return;
        sItem[rd & 1] = c2_item(p, rd, items);
        mbar_arrive(&item_full[rd & 1]);
      };
      publish(0);
      for (int rd = 0; ok; ++rd) {
        const C2Item own = sItem[rd & 1];
        if (own.b < 0) break;
        publish(rd + 1);
        ok = ok && mbar_wait(q_free, (rd & 1) ^ 1u, abort_flag, p.status, 0xC30);
        if (!ok) break;
        mbar_expect_tx(q_full, 2u * (uint32_t)(D / 64) * 128u * (uint32_t)(toks * G));
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            tma_load_3d(sQ + x * Tile::kQ + c * kScSub, &tmap_q, q_full, c * 64, own.kvh * G, own.q_row0 + own.q0 + x * toks);
      }
      if (!ok)
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------------------------------------------- heads of 256
// One query tile a CTA: its output takes half of TMEM, the query rows a quarter (as operands of the scores they would be read from shared
// memory once for 64 keys), two buffers of 64 score columns the rest.
//   warps 0..3     query rows to TMEM, softmax, a thread a row; P goes over its scores
//   warps 4..7     keys to bf16          warps 8..11   values to f16          (two buffers of each)
//   warps 14, 12   products: scores (of key tile j + 2 behind PV_j, whose P lies where they go), outputs
//   warp 13        pages by bulk copies, their scales
// Per 64 keys: products 512 clocks, exponentials 512, shared memory 1536 (512 for operands, 512 for the widened tiles, 512 for the codes).
// Measured 2700, the softmax thread's chain again (issue slots 48 %, tensor cores 40 %).  517 rows of 16 heads behind 4096 tokens: 56 us,
// 655 TFLOP/s (P through shared memory, two threads a row, one group of widening warps: 115).
constexpr int kWideThreads = 480, kWideKv = 64, kWidePages = 4, kWideRing = 8;

struct WideTile {
  static constexpr int D = 256;
  static constexpr int kSub = kWideKv * 128;                      // 64 tokens x 64 channels
  static constexpr int kK = (D / 64) * kSub, kV = D * 128;        // 64 tokens x D channels, D channels x 64 tokens
  static constexpr int kStage = kWideKv * D;
  static constexpr int kSmem = 2 * (kK + kV + 2 * kStage) + kWideRing * kWidePages * 8 + 256 + 1024;
};

__global__ void __launch_bounds__(kWideThreads, 1)
scaled_chunk_wide_kernel(const ScChunkParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using Tile = WideTile;
  constexpr int D = Tile::D;
  uint8_t* sK = smem;                                             // two buffers: D / 64 sub-tiles [64 tokens][64 channels]
  uint8_t* sV = sK + 2 * Tile::kK;                                // two buffers: [D channels][64 tokens]
  uint8_t* sStK = sV + 2 * Tile::kV;                              // two stages of pages as they come, keys and values
  uint8_t* sStV = sStK + 2 * Tile::kStage;
  float2* sScale = reinterpret_cast<float2*>(sStV + 2 * Tile::kStage);      // [kWideRing][4] (score factor, value exponent) of a page
  uint64_t* bars = reinterpret_cast<uint64_t*>(sScale + kWideRing * kWidePages);
  uint64_t* stage_full = bars;                                    // [keys, values][2] pages have come
  uint64_t* stage_free = bars + 4;                                // [keys, values][2] 4 warps
  uint64_t* k_full = bars + 8;                                    // [2] 4 warps
  uint64_t* k_free = bars + 10;                                   // [2] QK
  uint64_t* v_full = bars + 12;                                   // [2] 4 warps
  uint64_t* v_free = bars + 14;                                   // [2] PV
  uint64_t* s_full = bars + 16;                                   // [2]
  uint64_t* p_ready = bars + 18;                                  // [2] 4 warps
  uint64_t* pv_done = bars + 20;                                  // [2]
  uint64_t* q_ready = bars + 22;                                  // 4 warps
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 23);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  uint32_t* sFar = tmem_slot + 2;                                 // [kWideRing] whether a key tile has a far page

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.G, toks = kScRows / G;
  const int b = p.tile_seq[blockIdx.x], q0 = p.tile_q0[blockIdx.x], kvh = blockIdx.y, split = blockIdx.z;
  const int L = min(p.seq_lens[b], p.bt_cols * kScPg);
  const int q_row0 = p.query_start_loc[b], q_len = p.query_start_loc[b + 1] - q_row0;
  const int ctx0 = L - q_len;                                     // position of the chunk's first row
  const int kv_hi = min(L, ctx0 + min(q0 + toks, q_len));         // keys [.., kv_hi)
  const int first_page = p.window > 0 ? max(ctx0 + q0 - p.window + 1, 0) / kScPg : 0;
  const int all_kv = max((kv_hi - first_page * kScPg + kWideKv - 1) / kWideKv, 0), share = (all_kv + p.splits - 1) / p.splits;
  const int page0 = first_page + split * share * kWidePages;
  const int n_kv = min(max(all_kv - split * share, 0), share);

  if (threadIdx.x == 0) {
    for (int s = 0; s < 4; ++s) { mbar_init(&stage_full[s], 1); mbar_init(&stage_free[s], 4); }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], 4); mbar_init(&k_free[s], 1); mbar_init(&v_full[s], 4); mbar_init(&v_free[s], 1);
      mbar_init(&s_full[s], 1); mbar_init(&p_ready[s], 4); mbar_init(&pv_done[s], 1);
    }
    mbar_init(q_ready, 4);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 12) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;                               // scores (two times 64 columns), query rows (128), output (256)

  if (warp < 4) {
    // ------------------------------------------------------------------ softmax
    const int row = warp * 32 + lane;
    const uint32_t t_lane = (uint32_t)(warp * 32) << 16;
    const uint32_t tQ = tmem + 128 + t_lane, tO = tmem + 256 + t_lane;
    const int tok = q0 + row / G, head = kvh * G + row % G;
    const bool live = row < toks * G && tok < q_len;
    const __nv_bfloat16* q = p.q + (long long)(q_row0 + tok) * p.ldq + head * D;
#pragma unroll 4
    for (int c = 0; c < D / 32; ++c) {
      uint32_t v[16];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (live) x = *reinterpret_cast<const uint4*>(q + c * 32 + i * 8);
        v[4 * i] = x.x; v[4 * i + 1] = x.y; v[4 * i + 2] = x.z; v[4 * i + 3] = x.w;
      }
      tmem_st_32x32b_x16(tQ + c * 16, v);
    }
    tmem_st_wait();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_ready);
    // keys [start, end) are visible; rows that are not there see all, so that their warp need not mask, and are not stored
    const int pos = ctx0 + tok;
    const int end = live ? min(pos + 1, L) : 1 << 30;
    const int start = live && p.window > 0 ? pos - p.window + 1 : 0;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
#pragma unroll 1
    for (int j = 0; j < n_kv; ++j) {
      const int sb = j & 1;
      ok = mbar_wait(&s_full[sb], (j >> 1) & 1, abort_flag, p.status, 0xA00);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      tc_fence_after();
      const int kv0 = (page0 + j * kWidePages) * kScPg;
      const int hi = end - kv0, lo = start - kv0;
      const bool whole = __all_sync(0xffffffffu, hi >= kWideKv && lo <= 0);
      float2 f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = sScale[(j % kWideRing) * kWidePages + i];
      const uint32_t tS = tmem + sb * kWideKv + t_lane;
      auto output_there = [&] { return (bool)__all_sync(0xffffffffu, mbar_wait(&pv_done[sb ^ 1], ((j - 1) >> 1) & 1, abort_flag, p.status, 0xA01)); };
      ok = sFar[j % kWideRing] == 0 ? softmax_step<D, false>(tS, tS, tO, f, whole, hi, lo, j > 0, m, l, output_there)
                                    : softmax_step<D, true>(tS, tS, tO, f, whole, hi, lo, j > 0, m, l, output_there);
      if (!ok) break;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[sb]);
    }
    if (ok && n_kv > 0) ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[(n_kv - 1) & 1], ((n_kv - 1) >> 1) & 1, abort_flag, p.status, 0xA02));
    if (ok) {
      // ---- o / l, or this share's o and l
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const long long at = (long long)(q_row0 + tok) * p.Hq + head, at_part = ((long long)split * p.rows - p.first_row) * p.Hq + at;
      const bool part = p.splits > 1;
      tc_fence_after();
      store_outputs<D>(tO, n_kv == 0, inv, !live || (part && n_kv == 0) ? -1 : part ? at_part * D : (long long)(q_row0 + tok) * p.ldo + head * D, p.out, part ? p.part_o : nullptr, [] {});
      if (live) {
        if (part) p.part_ml[at_part] = make_float2(m, l);
        else if (p.ml) p.ml[at] = make_float2(m == -INFINITY ? 0.f : m, inv);
      }
    }
  } else if (warp < 8) {
    // ------------------------------------------------------------------ keys.  Eight neighbouring lanes take 64 bytes each of two rows, from
    // different sub-tiles: no two of their loads, and none of their stores, fall into the same banks.
    const int i8 = (threadIdx.x - 128) >> 5, sub = (lane >> 2) & 3, par = ((lane >> 2) & 1) ^ (lane >> 4), ch = (lane & 3) * 2;
    for (int j = 0; j < n_kv; ++j) {
      const int s = j & 1;
      const bool ok = mbar_wait(&stage_full[s], (j >> 1) & 1, abort_flag, p.status, 0xA10) &&
                      mbar_wait(&k_free[s], ((j >> 1) & 1) ^ 1u, abort_flag, p.status, 0xA11);
      if (!__all_sync(0xffffffffu, ok)) break;
#pragma unroll 4
      for (int k = 0; k < kWideKv / 8; ++k) {
        const int trow = (k * 4 + i8) * 2 + par, tsw = trow & 7;
        uint4 lo, hi;
        sc_widen16(*reinterpret_cast<const uint4*>(sStK + s * Tile::kStage + trow * D + sub * 64 + (lane & 3) * 16), lo, hi);
        uint8_t* rowp = sK + s * Tile::kK + sub * Tile::kSub + trow * 128;
        *reinterpret_cast<uint4*>(rowp + ((ch ^ tsw) << 4)) = f16_to_bf16(lo);
        *reinterpret_cast<uint4*>(rowp + (((ch + 1) ^ tsw) << 4)) = f16_to_bf16(hi);
      }
      fence_proxy_async();                                        // the tile for the products, and the pages read before they are copied over
      __syncwarp();
      if (lane == 0) { mbar_arrive(&k_full[s]); mbar_arrive(&stage_free[s]); }
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------------ values
    const int r = threadIdx.x - 256;
    for (int j = 0; j < n_kv; ++j) {
      const int s = j & 1;
      const bool ok = mbar_wait(&stage_full[2 + s], (j >> 1) & 1, abort_flag, p.status, 0xA12) &&
                      mbar_wait(&v_free[s], ((j >> 1) & 1) ^ 1u, abort_flag, p.status, 0xA13);
      if (!__all_sync(0xffffffffu, ok)) break;
      auto widen = [&](auto far) {                                // a far page: bf16; the usual loop stays free of that
#pragma unroll 4
        for (int k = 0; k < kWidePages * D / 128; ++k) {
          const int i = k * 128 + value_piece(r), pg = i / D, dim = i % D, col = output_column(dim), sw = col & 7, ch = pg * 2;
          const int left = L - (page0 + j * kWidePages + pg) * kScPg;       // tokens of the page; the others are cleared
          uint4 v = reinterpret_cast<const uint4*>(sStV + s * Tile::kStage)[i];
          if (left < kScPg) {
            uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int there = min(max(left - 4 * q, 0), 4);
              w[q] = there == 4 ? w[q] : (w[q] & ((1u << (8 * there)) - 1u));
            }
          }
          uint4 lo, hi;
          sc_widen16(v, lo, hi);
          if constexpr (decltype(far)::value) { lo = f16_to_bf16(lo); hi = f16_to_bf16(hi); }
          uint8_t* rowp = sV + s * Tile::kV + col * 128;
          *reinterpret_cast<uint4*>(rowp + ((ch ^ sw) << 4)) = lo;
          *reinterpret_cast<uint4*>(rowp + (((ch + 1) ^ sw) << 4)) = hi;
        }
      };
      if (sFar[j % kWideRing] == 0) widen(std::false_type{});
      else widen(std::true_type{});
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) { mbar_arrive(&v_full[s]); mbar_arrive(&stage_free[2 + s]); }
    }
  } else if (warp == 12 || warp == 14) {
    // ------------------------------------------------------------------ products (whole warps, one elected lane issues): warp 14 scores, warp 12
    // outputs, so that neither waits for the other's queue
    const uint32_t dK = desc_low(sK), dV = desc_low(sV), tQ = tmem + 128, tO = tmem + 256;
    auto wait = [&](uint64_t* bar, int j, uint32_t site) { return (bool)__all_sync(0xffffffffu, mbar_wait(bar + (j & 1), (j >> 1) & 1, abort_flag, p.status, site)); };
    if (warp == 14) {
      constexpr uint32_t kIdesc = make_idesc(kScRows, kWideKv, 1u);         // bf16
      if (__all_sync(0xffffffffu, mbar_wait(q_ready, 0, abort_flag, p.status, 0xA21)))
        for (int j = 0; j < n_kv; ++j) {
          // the product that read P out of these columns is done
          if (!wait(k_full, j, 0xA20) || (j >= 2 && !wait(pv_done, j - 2, 0xA24))) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
              umma_f16_ta(tmem + (j & 1) * kWideKv, tQ + ks * 8, dK + (j & 1) * (Tile::kK >> 4) + (ks >> 2) * (Tile::kSub >> 4) + 2 * (ks & 3), kIdesc,
                          ks > 0 ? 1u : 0u);
            umma_commit(&s_full[j & 1]);
            umma_commit(&k_free[j & 1]);
          }
          __syncwarp();
        }
    } else {
      constexpr uint32_t kIdesc = make_idesc(kScRows, D, 0u), kIdescFar = make_idesc(kScRows, D, 1u);      // f16; bf16, of two terms
      for (int j = 0; j < n_kv; ++j) {
        if (!wait(v_full, j, 0xA22) || !wait(p_ready, j, 0xA23)) break;
        tc_fence_after();
        const bool far = sFar[j % kWideRing] != 0;
        if (elect_one()) {
          const uint32_t tP = tmem + (j & 1) * kWideKv, bd = dV + (j & 1) * (Tile::kV >> 4);
          const uint32_t more = j > 0;
          if (!far) {
#pragma unroll
            for (int ks = 0; ks < kWideKv / 16; ++ks) umma_f16_ta(tO, tP + ks * 8, bd + 2 * ks, kIdesc, ks > 0 ? 1u : more);
          } else {
#pragma unroll
            for (int ks = 0; ks < kWideKv / 8; ++ks) umma_f16_ta(tO, tP + ks * 8, bd + 2 * (ks % 4), kIdescFar, ks > 0 ? 1u : more);
          }
          umma_commit(&pv_done[j & 1]);
          umma_commit(&v_free[j & 1]);
        }
        __syncwarp();
      }
    }
  } else {
    // ------------------------------------------------------------------ pages: lanes 0..3 keys, 8..11 values, entries and scales two tiles ahead
    const bool is_v = (lane & 8) != 0;
    const int n_pages = (L + kScPg - 1) / kScPg;
    const int* bt = p.block_tables + (long long)b * p.bt_ld;
    auto entry = [&](int j) {                                     // -1: behind the end or outside of the pool
      const int pg = page0 + j * kWidePages + (lane & 7);
      return lane < 16 && (lane & 7) < kWidePages && j < n_kv && pg < n_pages ? bt[pg] : -1;
    };
    auto scale_of = [&](int blk) {
      if ((unsigned)blk >= (unsigned)p.num_pages) return 1.f;
      return is_v ? p.v_scale[blk * p.vs_ld + kvh * p.vs_h] : p.k_scale[blk * p.ks_ld + kvh * p.ks_h];
    };
    const int newest = n_pages > 0 ? bt[n_pages - 1] : -1;
    int blk = entry(0), blk1 = entry(1);
    const float last = (unsigned)newest < (unsigned)p.num_pages ? p.v_scale[newest * p.vs_ld + kvh * p.vs_h] : 0.f;
    float sc = scale_of(blk);
    NearScales near;
    bool ok = true;
    for (int j = 0; j < n_kv; ++j) {
      const int blk2 = entry(j + 2), s = j & 1;
      const float sc1 = scale_of(blk1);
      const bool live = (unsigned)blk < (unsigned)p.num_pages;
      const uint32_t pages = __ballot_sync(0xffffffffu, live);
      const bool skip = lane < kWidePages && page0 + j * kWidePages + lane < n_pages && !live;
      const uint32_t skipped = __ballot_sync(0xffffffffu, skip);
      const long long at = ((long long)blk * p.Hkv + kvh) * (kScPg * D);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        ok = mbar_wait(&stage_free[2 * w + s], ((j >> 1) & 1) ^ 1u, abort_flag, p.status, 0xA30 + w);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        if (skipped) clear_pages<D>((w ? sStV : sStK) + s * Tile::kStage, skipped);
        if (lane == 0) sc_expect(&stage_full[2 * w + s], (uint32_t)__popc((pages >> (8 * w)) & 0xFFu) * (kScPg * D));
        __syncwarp();
        if (live && is_v == (w == 1))
          bulk_page((w ? sStV : sStK) + s * Tile::kStage + (lane & 7) * (kScPg * D), (w ? p.v_cache : p.k_cache) + at, kScPg * D, &stage_full[2 * w + s]);
        if (w == 0) {                                             // under the copies, as above; tile j - kWideRing is done: its keys left this stage long ago
          const float vs = __shfl_sync(0xffffffffu, sc, 8 + (lane & 7));
          if (j == 0) near.begin(pages >> 8 & 1 ? __shfl_sync(0xffffffffu, sc, 8) : 0.f, last);
          const bool far = __any_sync(0xffffffffu, live && is_v && near.far(sc));
          if (lane < kWidePages) sScale[(j % kWideRing) * kWidePages + lane] = skip ? skipped_page() : make_float2(p.scale_log2 * sc, (float)scale_exponent(vs));
          if (lane == 8) sFar[j % kWideRing] = far;
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(&stage_full[2 * w + s]);
      }
      if (!ok) break;
      blk = blk1; blk1 = blk2;
      sc = sc1;
    }
    if (!ok)
      for (int i = 0; i < 64; ++i) __nanosleep(1000);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------------------------------------------- weights
constexpr int kSwThreads = 320;        // producer, issuer, eight warps that add
constexpr int kSwStages = 2;           // query tiles in shared memory, score buffers in TMEM

ATLAS_DEVICE void st_cluster_f32(uint32_t addr, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;\n" ::"r"(addr), "f"(v) : "memory"); }

struct ScWeighParams {
  const uint8_t* k_cache; const float* k_scale; long long ks_ld; int ks_h;
  const int* block_tables; int bt_ld, bt_cols;
  const int* seq_lens; const int* query_start_loc;
  const int* tile_seq; const int* tile_k0;
  float scale_log2;
  int Hq, Hkv, G, window, num_pages;
  const float2* ml;
  float* weights; long long w_ld_b, w_ld_h; int width;
  status_t* status;
};

template <int D>
struct SwTile {
  static constexpr int kQ = (D / 64) * kScSub;                    // a query tile
  static constexpr int kSmem = (1 + kSwStages) * kQ + kSwStages * kScRows * 8 + 3 * kScRows * 4 + 128 + 1024;      // 101 KB for heads of 128: two CTAs
};

template <int D>
__global__ void __launch_bounds__(kSwThreads, D == 256 ? 1 : 2)
scaled_chunk_weigh_kernel(const __grid_constant__ CUtensorMap tmap_q, const ScWeighParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int kQ = SwTile<D>::kQ;
  uint8_t* sK = smem;                                              // D / 64 sub-tiles [128 tokens][64 channels], bf16
  uint8_t* sQ = sK + kQ;                                           // kSwStages x the same of query rows
  float* sM = reinterpret_cast<float*>(sQ + kSwStages * kQ);       // [stages][-M of 128 rows, 1 / l of 128 rows]
  float* sSum = sM + kSwStages * 2 * kScRows;
  float* sOwn = sSum + kScRows;                                    // [128] this CTA's sums
  float* sOther = sOwn + kScRows;                                  // [128] the other CTA's, in the first one
  uint64_t* bars = reinterpret_cast<uint64_t*>(sOther + kScRows);
  uint64_t* q_full = bars;                                         // [stages] the tile's bytes, its references
  uint64_t* q_empty = q_full + kSwStages;                          // [stages] QK done
  uint64_t* s_full = q_empty + kSwStages;                          // [stages]
  uint64_t* s_free = s_full + kSwStages;                           // [stages] 8 warps
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_free + kSwStages);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.G, toks = kScRows / G;
  const int part = blockIdx.x & 1, at = blockIdx.x >> 1;          // of a cluster of two: every other tile of rows
  const int b = p.tile_seq[at / p.Hkv], k0 = p.tile_k0[at / p.Hkv], kvh = at % p.Hkv;
  const int L = min(p.seq_lens[b], p.bt_cols * kScPg);
  const int q_row0 = p.query_start_loc[b], q_len = p.query_start_loc[b + 1] - q_row0;
  const int ctx0 = L - q_len;
  // rows that see some of the tokens [k0, k0 + 128): positions [k0, k0 + 127 + window)
  const int r_lo = max(k0 - ctx0, 0) / toks * toks + part * toks;
  const int r_hi = p.window > 0 ? min(q_len, k0 + kScRows - 1 + p.window - ctx0) : q_len;
  const int n_q = r_hi > r_lo ? (r_hi - r_lo + 2 * toks - 1) / (2 * toks) : 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kSwStages; ++s) { mbar_init(&q_full[s], 2); mbar_init(&q_empty[s], 1); mbar_init(&s_full[s], 1); mbar_init(&s_free[s], 8); }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) { tmem_alloc(tmem_slot, 256); tmem_relinquish(); }
  if (warp >= 2) {
    // the tokens' codes to bf16; tokens past the end are zero
    const int* bt = p.block_tables + (long long)b * p.bt_ld;
    for (int i = threadIdx.x - 64; i < kScRows * (D / 16); i += kSwThreads - 64) {
      const int trow = i / (D / 16), c = i % (D / 16), tsw = trow & 7, tok = k0 + trow;
      uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
      if (tok < L) {
        const int blk = bt[tok / kScPg];
        if (blk >= 0 && blk < p.num_pages)
          sc_widen16(*reinterpret_cast<const uint4*>(p.k_cache + (((long long)blk * p.Hkv + kvh) * kScPg + tok % kScPg) * D + c * 16), lo, hi);
      }
      uint32_t* w[2] = {reinterpret_cast<uint32_t*>(&lo), reinterpret_cast<uint32_t*>(&hi)};
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) w[a][e] = h2_to_bf2(w[a][e]);
      uint8_t* rowp = sK + (c >> 2) * kScSub + (trow >> 3) * 1024 + tsw * 128;
      const int ch = (c & 3) * 2;
      *reinterpret_cast<uint4*>(rowp + ((ch ^ tsw) << 4)) = lo;
      *reinterpret_cast<uint4*>(rowp + (((ch + 1) ^ tsw) << 4)) = hi;
    }
    // rows behind a tile's last whole token are never loaded: zeros
    for (int i = threadIdx.x - 64; i < kSwStages * (D / 64) * (kScRows - toks * G) * 8; i += kSwThreads - 64) {
      const int r = toks * G + (i >> 3) % (kScRows - toks * G), sub = (i >> 3) / (kScRows - toks * G);
      *reinterpret_cast<uint4*>(sQ + sub * kScSub + (r >> 3) * 1024 + (r & 7) * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async();
  }
  if (threadIdx.x < kScRows) sSum[threadIdx.x] = 0.f;
  tc_fence_before();
  cluster_sync_all();          // the other CTA runs, too: without rows of its own a CTA stores into it at once
  tc_fence_after();
  const uint32_t tS = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------------ producer: query rows as soon as the last product has read its buffer, and
    // their M and 1 / l, loaded a tile ahead, when the sums have (both of a tile, loaded then: 118 in place of 104 us for 2 x 3001 rows)
    bool ok = true;
    float2 x[kScRows / 32];
    auto references = [&](int j) {
      const int q0 = r_lo + j * 2 * toks;
#pragma unroll
      for (int i = 0; i < kScRows / 32; ++i) {
        const int r = i * 32 + lane, tok = q0 + r / G;
        x[i] = make_float2(INFINITY, 0.f);                         // a row that is not there adds 2^-inf * 0
        if (r < toks * G && tok < q_len) x[i] = p.ml[(long long)(q_row0 + tok) * p.Hq + kvh * G + r % G];
      }
    };
    if (n_q > 0) references(0);
    for (int j = 0; j < n_q; ++j) {
      const int s = j % kSwStages, q0 = r_lo + j * 2 * toks;
      ok = mbar_wait(&q_empty[s], ((j / kSwStages) & 1) ^ 1u, abort_flag, p.status, 0xB00);
      if (!__all_sync(0xffffffffu, ok)) break;
      if (lane == 0) {
        mbar_expect_tx(&q_full[s], (uint32_t)(D / 64) * 128u * (uint32_t)(toks * G));
#pragma unroll
        for (int c = 0; c < D / 64; ++c) tma_load_3d(sQ + s * kQ + c * kScSub, &tmap_q, &q_full[s], c * 64, kvh * G, q_row0 + q0);
      }
      ok = mbar_wait(&s_free[s], ((j / kSwStages) & 1) ^ 1u, abort_flag, p.status, 0xB01);
      if (!__all_sync(0xffffffffu, ok)) break;
#pragma unroll
      for (int i = 0; i < kScRows / 32; ++i) {
        sM[s * 2 * kScRows + i * 32 + lane] = -x[i].x;
        sM[s * 2 * kScRows + kScRows + i * 32 + lane] = x[i].y;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[s]);
      if (j + 1 < n_q) references(j + 1);
    }
    if (*abort_flag)
      for (int i = 0; i < 64; ++i) __nanosleep(1000);
  } else if (warp == 1) {
    // ------------------------------------------------------------------ products: S^T = K Q^T (the whole warp, one elected lane issues)
    constexpr uint32_t kIdesc = make_idesc(kScRows, kScRows, 1u);        // bf16 x bf16 -> f32
    const uint32_t dK = desc_low(sK), dQ = desc_low(sQ);
    for (int j = 0; j < n_q; ++j) {
      const int s = j % kSwStages;
      if (!__all_sync(0xffffffffu, mbar_wait(&q_full[s], (j / kSwStages) & 1, abort_flag, p.status, 0xB10))) break;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t at = (ks >> 2) * (kScSub >> 4) + 2 * (ks & 3);
          umma_f16_lo(tS + s * kScRows, dK + at, dQ + s * (kQ >> 4) + at, kIdesc, ks > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[s]);
        umma_commit(&q_empty[s]);
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------------ two threads a token, 64 rows each
    const int lane_group = warp & 3, half = (warp - 2) >> 2;
    const int trow = lane_group * 32 + lane, tok = k0 + trow;
    const uint32_t t_lane = (uint32_t)(lane_group * 32) << 16;
    float f = 0.f;
    bool skip = true;                                      // a token of a page outside of the pool gets no weight
    if (tok < L) {
      const int blk = p.block_tables[(long long)b * p.bt_ld + tok / kScPg];
      skip = blk < 0 || blk >= p.num_pages;
      if (!skip) f = p.scale_log2 * p.k_scale[blk * p.ks_ld + kvh * p.ks_h];
    }
    float total = 0.f;
    bool ok = true;
    for (int j = 0; j < n_q && ok; ++j) {
      const int s = j % kSwStages, q0 = r_lo + j * 2 * toks;
      ok = mbar_wait(&s_full[s], (j / kSwStages) & 1, abort_flag, p.status, 0xB20);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      tc_fence_after();
      // row r of the tile stands at position first + r / G: seen by tokens in (position - window, position]
      const int first = ctx0 + q0;
      const int there = min(toks, q_len - q0);             // rows behind them are another sequence's
      const bool all_seen = there == toks && k0 + kScRows - 1 <= first && (p.window == 0 || first + toks - 1 - p.window < k0);
      // columns of rows that see this lane's token
      const int c_lo = max(tok - first, 0) * G, c_hi = (p.window > 0 ? min(tok + p.window - first, there) : there) * G;
      const uint64_t f2 = pair2(f, f);
      uint64_t sum2 = 0;
#pragma unroll 2
      for (int c = half * 64; c < half * 64 + 64; c += 32) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(tS + s * kScRows + t_lane + c, r);
        const float4* m4 = reinterpret_cast<const float4*>(sM + s * 2 * kScRows + c);
        const float4* l4 = reinterpret_cast<const float4*>(sM + s * 2 * kScRows + kScRows + c);
        const uint32_t seen = all_seen ? 0xffffffffu : bits_below(c_hi - c) & ~bits_below(c_lo - c);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 m = m4[i / 4], l = l4[i / 4];
          float2 a = unpair2(fma2(pair2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), f2, pair2(m.x, m.y)));
          float2 b2 = unpair2(fma2(pair2(__uint_as_float(r[i + 2]), __uint_as_float(r[i + 3])), f2, pair2(m.z, m.w)));
          a.x = fast_exp2(a.x); a.y = fast_exp2(a.y); b2.x = fast_exp2(b2.x); b2.y = fast_exp2(b2.y);
          if (!all_seen) {                                  // the same for all lanes
            a.x = (seen >> i) & 1u ? a.x : 0.f;
            a.y = (seen >> (i + 1)) & 1u ? a.y : 0.f;
            b2.x = (seen >> (i + 2)) & 1u ? b2.x : 0.f;
            b2.y = (seen >> (i + 3)) & 1u ? b2.y : 0.f;
          }
          sum2 = fma2(pair2(a.x, a.y), pair2(l.x, l.y), sum2);
          sum2 = fma2(pair2(b2.x, b2.y), pair2(l.z, l.w), sum2);
        }
      }
      const float2 sums = unpair2(sum2);
      total += sums.x + sums.y;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_free[s]);
    }
    if (skip) total = 0.f;
    if (half == 1) sSum[trow] = total;
    asm volatile("bar.sync 1, 256;\n" ::: "memory");
    if (half == 0) {
      total += sSum[trow];
      if (part == 0) sOwn[trow] = total;
      else st_cluster_f32(cluster_map_shared(smem_u32(sOther + trow), 0), total);
    }
  }
  tc_fence_before();
  cluster_sync_all();
  if (part == 0 && threadIdx.x < kScRows && !*abort_flag) {
    const int tok = k0 + (int)threadIdx.x;
    if (tok < L && tok < p.width) p.weights[b * p.w_ld_b + kvh * p.w_ld_h + tok] += sOwn[threadIdx.x] + sOther[threadIdx.x];
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tS, 256);
  }
}

}  // namespace atlas

using namespace atlas;

namespace {

// Q as [tokens][heads][channels]: boxes of 64 channels x G heads x 128 / G tokens, rows of 128 bytes, row = token * G + head
int query_map(CUtensorMap* m, const void* q, long long ldq, int total_tokens, int Hq, int G, int D) {
  EncodeTiledFn enc = tc_encode_fn();
  if (!enc) return -10;
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)Hq, (cuuint64_t)total_tokens};
  cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)ldq * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)(kScRows / G)};
  cuuint32_t estr[3] = {1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : -11;
}

template <typename Kern>
int launch_pairs(Kern kern, int smem, int blocks, const CUtensorMap& tq, const ScChunkParams& p, int items, cudaStream_t st) {
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem) != cudaSuccess) return -20;
  kern<<<blocks, kC2Threads, smem, st>>>(tq, p, items);
  return cudaGetLastError() == cudaSuccess ? 0 : -20;
}

int launch_weigh(void (*kern)(CUtensorMap, ScWeighParams), int smem, unsigned blocks, const CUtensorMap& tq, const ScWeighParams& p, cudaStream_t st) {
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem) != cudaSuccess) return -20;
  if (launch_chain_cluster(false, 2, kern, dim3(blocks), dim3(kSwThreads), smem, st, tq, p) != cudaSuccess) { cudaGetLastError(); return -20; }
  return 0;
}

int launch_wide(dim3 grid, const ScChunkParams& p, cudaStream_t st) {
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(scaled_chunk_wide_kernel), WideTile::kSmem) != cudaSuccess) return -20;
  scaled_chunk_wide_kernel<<<grid, kWideThreads, WideTile::kSmem, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : -20;
}

}  // namespace

// Rows of chunk sequences: `tiles` query tiles of 128 / G tokens (heads of 64 and 128: pairs of tiles), each (sequence, first token in its
// chunk); `ml` (or null) gets every row's reference and 1 / l.  `splits` > 1: part_o [splits][rows][Hq][D] and part_ml [splits][rows][Hq][2]
// for the rows from first_row on, the chunks'.  With `weights`, tiles of 128 cached tokens follow, each (sequence, first token), whose sums grow
// by the rows' softmax weights.  Arguments as one record (see kv_scaled.cu).  -1: sizes or alignment outside of what the kernels take.
struct ChunkRecord {
  const void* q; long long ldq; void* out; long long ldo; const void* k_cache; const void* v_cache;
  const float* ks; long long ks_ld, ks_h; const float* vs; long long vs_ld, vs_h;
  const int* tables; long long bt_ld, bt_cols; const int* seq_lens; const int* starts;
  const int* tile_seq; const int* tile_q0; long long tiles, total_tokens, Hq, Hkv, D, window, num_pages; float* ml; long long splits, first_row; float* part_o; float* part_ml;
  const int* key_seq; const int* key_k0; long long key_tiles; float* weights; long long w_ld_b, w_ld_h, width, sms; double scale; void* status;
  void* stream;
};
extern "C" int atlas_attn_scaled_chunk(const void* record) {
  const ChunkRecord& r = *static_cast<const ChunkRecord*>(record);
  const int D = (int)r.D;
  if (r.tiles <= 0) return 0;
  if ((D != 64 && D != 128 && D != 256) || r.Hkv <= 0 || r.Hkv > 65535 || r.Hq < r.Hkv || r.Hq % r.Hkv || r.Hq / r.Hkv > kScRows) return -1;
  if ((reinterpret_cast<uintptr_t>(r.q) & 15) || r.ldq % 8 || r.ldo % 8 || (reinterpret_cast<uintptr_t>(r.out) & 15)) return -1;
  if ((reinterpret_cast<uintptr_t>(r.k_cache) | reinterpret_cast<uintptr_t>(r.v_cache)) & 15) return -1;
  if (!(r.scale >= 0x1p-60 && r.scale <= 0x1p60)) return -1;      // scores are masked, and the largest is taken, before their factor is applied
  if (r.bt_cols > (1 << 25) || r.window < 0 || r.window > (1 << 29) || r.tiles > 0x7fffffffll || r.total_tokens > 0x7fffffffll || (r.weights && !r.ml)) return -1;
  if (r.splits < 1 || r.splits > 65535 || (r.splits > 1 && (!r.part_o || !r.part_ml)) || r.first_row < 0 || r.first_row >= r.total_tokens) return -1;
  const int Hq = (int)r.Hq, Hkv = (int)r.Hkv, G = Hq / Hkv;
  CUtensorMap tq;
  if (int rc = query_map(&tq, r.q, r.ldq, (int)r.total_tokens, Hq, G, D)) return rc;
  const float scale_log2 = (float)(r.scale * 1.4426950408889634);
  status_t* status = (status_t*)r.status;
  cudaStream_t st = (cudaStream_t)r.stream;
  ScChunkParams p{(const __nv_bfloat16*)r.q, r.ldq, (__nv_bfloat16*)r.out, r.ldo, (const uint8_t*)r.k_cache, (const uint8_t*)r.v_cache, r.ks, r.vs, r.ks_ld, r.vs_ld, (int)r.ks_h,
                  (int)r.vs_h, r.tables, (int)r.bt_ld, (int)r.bt_cols, r.seq_lens, r.starts, r.tile_seq, r.tile_q0, scale_log2, Hq, Hkv, G,
                  (int)r.window, (int)r.num_pages, reinterpret_cast<float2*>(r.ml), (int)r.splits, (int)r.first_row,
                  (int)(r.total_tokens - r.first_row), r.part_o,
                  reinterpret_cast<float2*>(r.part_ml), status};
  int rc;
  if (D <= 128) {
    const long long items = r.tiles * Hkv * r.splits;
    if (items > 0x3fffffffll) return -1;
    const int blocks = (int)(items < r.sms ? items : r.sms);
    if (D == 64) rc = launch_pairs(scaled_chunk2_kernel<64>, C2Tile<64>::kSmem, blocks, tq, p, (int)items, st);
    else rc = launch_pairs(scaled_chunk2_kernel<128>, C2Tile<128>::kSmem, blocks, tq, p, (int)items, st);
  } else rc = launch_wide(dim3((unsigned)r.tiles, Hkv, (unsigned)r.splits), p, st);
  if (rc) return rc;
  if (r.splits > 1) {
    const unsigned blocks = (unsigned)(((r.total_tokens - r.first_row) * Hq + 7) / 8);
    if (D == 64) scaled_chunk_join_kernel<64><<<blocks, 256, 0, st>>>(p);
    else if (D == 128) scaled_chunk_join_kernel<128><<<blocks, 256, 0, st>>>(p);
    else scaled_chunk_join_kernel<256><<<blocks, 256, 0, st>>>(p);
    if (cudaGetLastError() != cudaSuccess) return -20;
  }
  if (!r.weights || r.key_tiles <= 0) return 0;
  ScWeighParams w{(const uint8_t*)r.k_cache, r.ks, r.ks_ld, (int)r.ks_h, r.tables, (int)r.bt_ld, (int)r.bt_cols, r.seq_lens, r.starts, r.key_seq,
                  r.key_k0, scale_log2, Hq, Hkv, G, (int)r.window, (int)r.num_pages, reinterpret_cast<const float2*>(r.ml), r.weights, r.w_ld_b,
                  r.w_ld_h, (int)r.width, status};
  const long long keys = 2 * r.key_tiles * Hkv;
  if (keys > 0x7fffffffll) return -1;
  if (D == 64) return launch_weigh(scaled_chunk_weigh_kernel<64>, SwTile<64>::kSmem, (unsigned)keys, tq, w, st);
  if (D == 128) return launch_weigh(scaled_chunk_weigh_kernel<128>, SwTile<128>::kSmem, (unsigned)keys, tq, w, st);
  return launch_weigh(scaled_chunk_weigh_kernel<256>, SwTile<256>::kSmem, (unsigned)keys, tq, w, st);
}

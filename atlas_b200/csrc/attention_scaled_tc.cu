// Chunk attention over the FP8 cache with a power-of-two scale per (page, head), on the 5th-generation tensor cores, and the softmax weight
// that each cached token got from a chunk's rows.
//
// As in attention_scaled.cu the codes are the operands and the scales live in the exponent: s_j = f q . k^_j with f = softmax scale * log2(e) *
// 2^(row's own power) * key page's scale, p_j = 2^(s_j + ev - M) in f16, o = sum p_j v^_j / sum p_j 2^-ev.  A page covers 16 score columns, so
// f and ev - M are constants of a multiply-add over them, and a page's largest score is found before they are applied.
//
// scaled_chunk_kernel: one CTA per (128 query rows, key head); the G query heads of a key head are packed into the rows (row = token * G +
// head), so that a page is fetched and widened once for all of them.
//   warp 0       Q tile by TMA; the pages of each key tile (cp.async.bulk) and their scales, a tile of block-table entries ahead
//   warp 1       tcgen05.mma: S_j = Q K_j^T into one of two score buffers, O += P_j V_j; QK_{j+1} goes before PV_j
//   warps 2..5   e4m3 -> f16, into the 128-byte-swizzled K-major layout (values are stored with tokens along rows already)
//   warps 6..13  softmax, two threads a row; O is rescaled in TMEM only when a row's maximum has passed its reference by 2^8
//
// scaled_chunk_weigh_kernel: one CTA per (128 cached tokens, key head), rows of the chunk go by.  S^T = K Q^T in bf16 (an e4m3 number is one
// exactly, and Q stays as it is): a TMEM lane is a token, so that the sum over rows and heads is a register's sum, with no atomics.
#include "common.cuh"
#include "host_api.h"
#include "tc_util.cuh"

namespace atlas {

constexpr int kScRows = 128;
constexpr int kScPg = 16;
constexpr int kScThreads = 448;
constexpr int kScSub = 16 * 1024;                 // 128 rows x 64 16-bit numbers
constexpr int kScRingTiles = 8;                   // key tiles whose page scales are kept

template <int D>
struct ScTile {
  static constexpr int kKv = D <= 128 ? 128 : 64;                // keys of a tile: 256-wide heads would not fit twice that
  static constexpr int kPages = kKv / kScPg;
  static constexpr int kKSub = kKv * 128, kVSub = D * 128;
  static constexpr int kPageBytes = kScPg * D;
  static constexpr int kStageBytes = 2 * kPages * kPageBytes;
  static constexpr int kStages = D <= 128 ? 3 : 2;
  static constexpr int kTiles = (D / 64) * (kScSub + kKSub) + (kKv / 64) * (kVSub + kScSub);
  static constexpr int kSmem = kTiles + kStages * kStageBytes + 2048 + 1024;
};

struct ScChunkParams {
  __nv_bfloat16* out; long long ldo;
  const uint8_t* k_cache; const uint8_t* v_cache;
  const float* k_scale; const float* v_scale; long long ks_ld, vs_ld; int ks_h, vs_h;
  const int* block_tables; int bt_ld, bt_cols;
  const int* seq_lens; const int* query_start_loc;
  const int* tile_seq; const int* tile_q0;
  float scale_log2;
  int Hq, Hkv, G, window, num_pages;
  float2* ml;                                     // [rows of the step][Hq] (M, 1 / l) or null
  status_t* status;
};

ATLAS_DEVICE void sc_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
ATLAS_DEVICE uint32_t sc_e4m3x2(uint32_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(r) : "h"((uint16_t)v));
  return r;
}
ATLAS_DEVICE uint32_t sc_h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
ATLAS_DEVICE void sc_widen16(const uint4 v, uint4& lo, uint4& hi) {
  lo.x = sc_e4m3x2(v.x); lo.y = sc_e4m3x2(v.x >> 16); lo.z = sc_e4m3x2(v.y); lo.w = sc_e4m3x2(v.y >> 16);
  hi.x = sc_e4m3x2(v.z); hi.y = sc_e4m3x2(v.z >> 16); hi.z = sc_e4m3x2(v.w); hi.w = sc_e4m3x2(v.w >> 16);
}
ATLAS_DEVICE uint32_t h2_to_bf2(uint32_t v) {      // e4m3 numbers: exact in both
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
  return pack_bf16x2(f.x, f.y);
}
ATLAS_DEVICE int scale_exponent(float s) { return (int)((__float_as_uint(s) >> 23) & 255u) - 127; }
ATLAS_DEVICE float exact_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

template <int D>
__global__ void __launch_bounds__(kScThreads, 1)
scaled_chunk_kernel(const __grid_constant__ CUtensorMap tmap_q, const ScChunkParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using Tile = ScTile<D>;
  constexpr int kKv = Tile::kKv, kPages = Tile::kPages, kStages = Tile::kStages, kStageBytes = Tile::kStageBytes;
  constexpr int kPageBytes = Tile::kPageBytes, kKSub = Tile::kKSub, kVSub = Tile::kVSub;
  uint8_t* sQ = smem;                              // D / 64 sub-tiles [128 rows][64 channels]
  uint8_t* sK = sQ + (D / 64) * kScSub;            // D / 64 sub-tiles [tokens][64 channels]
  uint8_t* sV = sK + (D / 64) * kKSub;             // kKv / 64 sub-tiles [channels][64 tokens]
  uint8_t* sP = sV + (kKv / 64) * kVSub;           // kKv / 64 sub-tiles [128 rows][64 tokens]
  uint8_t* sStage = smem + Tile::kTiles;           // kStages x (K pages, V pages)
  float2* sScale = reinterpret_cast<float2*>(sStage + kStages * kStageBytes);      // [kScRingTiles][8] (key scale, value exponent)
  float* sRow = reinterpret_cast<float*>(sScale + kScRingTiles * 8);               // [128] score factor of a row
  uint64_t* bars = reinterpret_cast<uint64_t*>(sRow + kScRows);
  uint64_t* q_full = bars;
  uint64_t* stg_full = bars + 1;                   // [kStages]
  uint64_t* stg_empty = stg_full + kStages;        // [kStages] 4 converter warps
  uint64_t* k_ready = stg_empty + kStages;         // 4 converter warps
  uint64_t* k_free = k_ready + 1;                  // QK done
  uint64_t* v_ready = k_ready + 2;                 // 4 converter warps
  uint64_t* pv_done = k_ready + 3;                 // V tile, P tile and O are free
  uint64_t* s_full = k_ready + 4;                  // [2]
  uint64_t* s_free = k_ready + 6;                  // [2] 8 softmax warps
  uint64_t* p_ready = k_ready + 8;                 // 8 softmax warps
  uint64_t* q_conv = k_ready + 9;                  // 8 softmax warps
  uint64_t* x_ready = k_ready + 10;                // [2 parities][4 row groups]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(k_ready + 18);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.G, tok_per_tile = kScRows / G;
  const int b = p.tile_seq[blockIdx.x], q0 = p.tile_q0[blockIdx.x], kvh = blockIdx.y;
  const int L = min(p.seq_lens[b], p.bt_cols * kScPg);
  const int q_row0 = p.query_start_loc[b], q_len = p.query_start_loc[b + 1] - q_row0;
  const int ctx0 = L - q_len;                                   // position of the chunk's first row
  const int last_tok = min(q0 + tok_per_tile, q_len) - 1;
  const int kv_hi = min(L, ctx0 + last_tok + 1);                // keys [.., kv_hi)
  const int page0 = p.window > 0 ? max(ctx0 + q0 - p.window + 1, 0) / kScPg : 0;
  const int base = page0 * kScPg;                               // first key of tile 0
  const int n_kv = max((kv_hi - base + kKv - 1) / kKv, 0);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < kStages; ++s) { mbar_init(&stg_full[s], 1); mbar_init(&stg_empty[s], 4); }
    for (int s = 0; s < 2; ++s) { mbar_init(&s_full[s], 1); mbar_init(&s_free[s], 8); }
    mbar_init(k_ready, 4); mbar_init(k_free, 1); mbar_init(v_ready, 4); mbar_init(pv_done, 1); mbar_init(p_ready, 8);
    mbar_init(q_conv, 8);
    for (int s = 0; s < 8; ++s) mbar_init(&x_ready[s], 2);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  if (warp == 0 && lane == 0) tma_prefetch_desc(&tmap_q);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t tS = tmem_base, tO = tmem_base + 2 * kKv, tX = tO + D;

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    if (lane == 0) {
      mbar_expect_tx(q_full, (uint32_t)(D / 64) * 128u * (uint32_t)(tok_per_tile * G));
#pragma unroll
      for (int s = 0; s < D / 64; ++s) tma_load_3d(sQ + s * kScSub, &tmap_q, q_full, s * 64, kvh * G, q_row0 + q0);
    }
    const int* bt = p.block_tables + (long long)b * p.bt_ld;
    const int n_pages = (L + kScPg - 1) / kScPg;
    const int pi = lane & 7;                           // lanes 0..7 fetch key pages, 8..15 value pages, the first kPages of each
    const bool is_v = (lane & 8) != 0;
    auto entry = [&](int j) {                          // block and scale of this lane's page of tile j
      const int pg = page0 + j * kPages + pi;
      int blk = lane < 16 && pi < kPages && pg < n_pages ? bt[pg] : -1;
      return blk >= p.num_pages ? -1 : blk;
    };
    auto scale_of = [&](int blk) {
      if (blk < 0) return 1.f;
      return is_v ? p.v_scale[blk * p.vs_ld + kvh * p.vs_h] : p.k_scale[blk * p.ks_ld + kvh * p.ks_h];
    };
    int blk_next = entry(0);
    float sc_next = scale_of(blk_next);
    uint32_t stage = 0, phase = 0;
    bool ok = true;
    for (int j = 0; j < n_kv && ok; ++j) {
      const int blk = blk_next;
      const float sc = sc_next;
      if (j + 1 < n_kv) { blk_next = entry(j + 1); sc_next = scale_of(blk_next); }
      if (lane == 0) ok = mbar_wait(&stg_empty[stage], phase ^ 1u, abort_flag, p.status, 0xA00);
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      if (!ok) break;
      const float vs = __shfl_sync(0xffffffffu, sc, 8 + (lane & 7));
      if (lane < kPages) sScale[(j % kScRingTiles) * 8 + lane] = make_float2(sc, (float)scale_exponent(vs));
      const uint32_t live = __popc(__ballot_sync(0xffffffffu, blk >= 0));
      __syncwarp();
      if (lane == 0) mbar_expect_tx(&stg_full[stage], live * (uint32_t)kPageBytes);
      __syncwarp();
      if (blk >= 0) {
        const long long page = (long long)blk * p.Hkv + kvh;
        uint8_t* dst = sStage + stage * kStageBytes + ((is_v ? kPages : 0) + pi) * kPageBytes;
        sc_bulk(dst, (is_v ? p.v_cache : p.k_cache) + page * kPageBytes, kPageBytes, &stg_full[stage]);
      }
      if (++stage == kStages) { stage = 0; phase ^= 1u; }
    }
    if (!ok)
      for (int i = 0; i < 64; ++i) __nanosleep(1000);
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t kIdescS = make_idesc(kScRows, kKv, 0u), kIdescO = make_idesc(kScRows, D, 0u);     // f16 x f16 -> f32
      const uint32_t aQ = smem_u32(sQ), aK = smem_u32(sK), aV = smem_u32(sV), aP = smem_u32(sP);
      bool ok = mbar_wait(q_conv, 0, abort_flag, p.status, 0xA10);
      auto issue_pv = [&](int i) -> bool {
        if (!mbar_wait(p_ready, i & 1, abort_flag, p.status, 0xA12)) return false;
        if (!mbar_wait(v_ready, i & 1, abort_flag, p.status, 0xA13)) return false;
        tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < kKv / 16; ++ks) {
          const uint64_t ad = make_smem_desc_sw128(aP + (ks >> 2) * kScSub) + 2 * (ks & 3);
          const uint64_t bd = make_smem_desc_sw128(aV + (ks >> 2) * kVSub) + 2 * (ks & 3);
          umma_f16(tO, ad, bd, kIdescO, (i > 0 || ks > 0) ? 1u : 0u);
        }
        umma_commit(pv_done);
        return true;
      };
      for (int j = 0; j < n_kv && ok; ++j) {
        const int sb = j & 1;
        if (!mbar_wait(k_ready, j & 1, abort_flag, p.status, 0xA14)) { ok = false; break; }
        if (!mbar_wait(&s_free[sb], ((j >> 1) & 1) ^ 1u, abort_flag, p.status, 0xA15)) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint64_t ad = make_smem_desc_sw128(aQ + (ks >> 2) * kScSub) + 2 * (ks & 3);
          const uint64_t bd = make_smem_desc_sw128(aK + (ks >> 2) * kKSub) + 2 * (ks & 3);
          umma_f16(tS + sb * kKv, ad, bd, kIdescS, ks > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[sb]);
        umma_commit(k_free);
        if (j > 0) ok = issue_pv(j - 1);
      }
      if (ok && n_kv > 0) issue_pv(n_kv - 1);
    }
  } else if (warp < 6) {
    // ------------------------------------------------------------------ converters
    const int r = threadIdx.x - 64;
    bool ok = true;
    auto conv_k = [&](int j) -> bool {
      const int s = j % kStages;
      if (!mbar_wait(&stg_full[s], (j / kStages) & 1, abort_flag, p.status, 0xA21)) return false;
      if (j > 0 && !mbar_wait(k_free, (j - 1) & 1, abort_flag, p.status, 0xA22)) return false;
      const int kv0 = base + j * kKv;
      const uint4* src = reinterpret_cast<const uint4*>(sStage + s * kStageBytes);
      // consecutive threads take consecutive 16-byte pieces: piece i = token i / (D / 16), channels (i % (D / 16)) * 16 ..
#pragma unroll
      for (int k8 = 0; k8 < kKv * (D / 16) / 128; ++k8) {
        const int i = k8 * 128 + r;
        const int trow = i / (D / 16), c = i % (D / 16), tsw = trow & 7;
        uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
        if (kv0 + trow < L) sc_widen16(src[i], lo, hi);
        uint8_t* rowp = sK + (c >> 2) * kKSub + (trow >> 3) * 1024 + tsw * 128;
        const int ch = (c & 3) * 2;
        *reinterpret_cast<uint4*>(rowp + ((ch ^ tsw) << 4)) = lo;
        *reinterpret_cast<uint4*>(rowp + (((ch + 1) ^ tsw) << 4)) = hi;
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(k_ready);
      return true;
    };
    auto conv_v = [&](int j) -> bool {
      const int s = j % kStages;
      const int kv0 = base + j * kKv;
      const uint8_t* stg = sStage + s * kStageBytes + kPages * kPageBytes;
      if (j > 0 && !mbar_wait(pv_done, (j - 1) & 1, abort_flag, p.status, 0xA23)) return false;
#pragma unroll
      for (int it = 0; it < D * kPages / 128; ++it) {
        const int i = it * 128 + r;
        const int pg = i / D, dim = i % D, sw = dim & 7;
        const int t0 = kv0 + pg * kScPg;
        uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
        if (t0 < L) {
          uint4 v = *reinterpret_cast<const uint4*>(stg + pg * kPageBytes + dim * kScPg);
          if (t0 + kScPg > L) {                       // the sequence ends inside this page
            uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int left = min(max(L - t0 - 4 * q, 0), 4);
              w[q] = left == 4 ? w[q] : (w[q] & ((1u << (8 * left)) - 1u));
            }
          }
          sc_widen16(v, lo, hi);
        }
        uint8_t* rowp = sV + (pg >> 2) * kVSub + (dim >> 3) * 1024 + sw * 128;
        const int ch = (pg & 3) * 2;
        *reinterpret_cast<uint4*>(rowp + ((ch ^ sw) << 4)) = lo;
        *reinterpret_cast<uint4*>(rowp + (((ch + 1) ^ sw) << 4)) = hi;
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) { mbar_arrive(v_ready); mbar_arrive(&stg_empty[s]); }
      return true;
    };
    if (n_kv > 0) ok = conv_k(0);
    for (int j = 0; j < n_kv && ok; ++j) {
      if (j + 1 < n_kv) ok = conv_k(j + 1);
      if (ok) ok = conv_v(j);
    }
  } else {
    // ------------------------------------------------------------------ softmax, two threads a row
    const int lane_group = warp & 3;                             // TMEM lanes 32 * (warp % 4) ..
    const int half = (warp - 6) >> 2;
    constexpr int HC = kKv / 2, HO = D / 2, HP = HC / kScPg;     // score columns, output columns and pages of a thread
    const int col0 = half * HC, ocol0 = half * HO;
    const int row = lane_group * 32 + lane;
    const uint32_t t_lane = (uint32_t)(lane_group * 32) << 16;
    bool ok = mbar_wait(q_full, 0, abort_flag, p.status, 0xA20);
    if (ok) {
      // Q to f16 in place: a row's largest magnitude to [2^13, 2^14), which keeps every bf16 number of it; two neighbouring lanes a row
      const int i = threadIdx.x - 192, r = i >> 1, part = i & 1, rsw = r & 7;
      constexpr int CH = D / 16;                                 // 16-byte chunks of a thread
      uint8_t* rowp = sQ + (r >> 3) * 1024 + rsw * 128;
      auto at = [&](int c) { return reinterpret_cast<uint4*>(rowp + (c >> 3) * kScSub + (((c & 7) ^ rsw) << 4)); };
      float amax = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const uint4 v = *at(2 * c + part);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[e]));
          amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      const int e2 = min(max(13 - ((int)(__float_as_uint(amax) >> 23) - 127), -100), 100);
      const float up = exact_pow2(e2);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        uint4* q4 = at(2 * c + part);
        uint4 v = *q4;
        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[e]));
          w[e] = sc_h2(f.x * up, f.y * up);
        }
        *q4 = v;
      }
      if (part == 0) sRow[r] = p.scale_log2 * exact_pow2(-e2);
      fence_proxy_async();
    }
    asm volatile("bar.sync 1, 256;\n" ::: "memory");             // the row factors, all softmax warps
    __syncwarp();
    if (lane == 0) mbar_arrive(q_conv);
    const float rf = sRow[row];
    int xn = 0;
    // one value per thread to the other thread of its row, through a TMEM column of the row's lane; slots alternate
    auto exchange = [&](float mine, float& other) -> bool {
      const int par = xn & 1;
      uint64_t* xb = &x_ready[par * 4 + lane_group];
      tmem_st_32x32b_x1(tX + t_lane + par * 2 + half, __float_as_uint(mine));
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(xb);
      if (!mbar_wait(xb, (xn >> 1) & 1, abort_flag, p.status, 0xA33)) return false;
      tc_fence_after();
      uint32_t o;
      tmem_ld_32x32b_x1(tX + t_lane + par * 2 + (half ^ 1), o);
      tmem_ld_wait();
      other = __uint_as_float(o);
      ++xn;
      return true;
    };
    const int tok = q0 + row / G;
    const int head = kvh * G + row % G;
    const bool row_live = row < tok_per_tile * G && tok < q_len;
    const int pos = ctx0 + tok;
    const int lo_key = p.window > 0 ? pos - p.window + 1 : 0;
    float m = -INFINITY, l = 0.f;
    const int sw = row & 7;
    uint8_t* prow = sP + (col0 >> 6) * kScSub + (row >> 3) * 1024 + sw * 128;
    const int pch = (col0 >> 3) & 7;
    for (int j = 0; j < n_kv && ok; ++j) {
      const int sb = j & 1, kv0 = base + j * kKv;
      if (!mbar_wait(&s_full[sb], (j >> 1) & 1, abort_flag, p.status, 0xA30)) { ok = false; break; }
      tc_fence_after();
      const int vis = row_live ? min(pos + 1, L) - kv0 : 0;      // columns [lo, vis) of this tile are visible
      const int low = lo_key - kv0;
      uint32_t sr[HC / 32][32];
#pragma unroll
      for (int c = 0; c < HC / 32; ++c) tmem_ld_32x32b_x32(tS + sb * kKv + t_lane + col0 + c * 32, sr[c]);
      float2 ps[HP];                                              // score factor and value exponent of a page
#pragma unroll
      for (int q = 0; q < HP; ++q) {
        const float2 x = sScale[(j % kScRingTiles) * 8 + half * HP + q];
        ps[q] = make_float2(rf * x.x, x.y);
      }
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_free[sb]);
      const bool full = __all_sync(0xffffffffu, vis >= col0 + HC && low <= col0);
      if (!full) {
#pragma unroll
        for (int c = 0; c < HC / 32; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (col0 + c * 32 + i >= vis || col0 + c * 32 + i < low) sr[c][i] = 0xff800000u;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int q = 0; q < HP; ++q) {
        float a = -INFINITY, z = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          a = fmaxf(a, __uint_as_float(sr[q >> 1][(q & 1) * 16 + i]));
          z = fmaxf(z, __uint_as_float(sr[q >> 1][(q & 1) * 16 + i + 1]));
        }
        mx = fmaxf(mx, fmaf(fmaxf(a, z), ps[q].x, ps[q].y));
      }
      float mx_other;
      if (!exchange(mx, mx_other)) { ok = false; break; }
      mx = fmaxf(mx, mx_other);
      float m_new = m, alpha = 1.f;
      if (mx > m + 8.f) {
        m_new = mx;
        alpha = (m == -INFINITY) ? 0.f : fast_exp2(m - mx);
      }
      if (j > 0) {
        if (!mbar_wait(pv_done, (j - 1) & 1, abort_flag, p.status, 0xA31)) { ok = false; break; }
        tc_fence_after();
        if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
          for (int c = 0; c < HO / 32; ++c) {
            uint32_t r[32];
            tmem_ld_32x32b_x32(tO + t_lane + ocol0 + c * 32, r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
            tmem_st_32x32b_x32(tO + t_lane + ocol0 + c * 32, r);
          }
          tmem_st_wait();
        }
      }
      const float mref = (m_new == -INFINITY) ? 0.f : m_new;
      float sum = 0.f;
#pragma unroll
      for (int q = 0; q < HP; ++q) {
        const float f = ps[q].x, add = ps[q].y - mref;
        float s0 = 0.f, s1 = 0.f;
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float e0 = fast_exp2(fmaf(__uint_as_float(sr[q >> 1][(q & 1) * 16 + i]), f, add));
          const float e1 = fast_exp2(fmaf(__uint_as_float(sr[q >> 1][(q & 1) * 16 + i + 1]), f, add));
          s0 += e0;
          s1 += e1;
          w[i >> 1] = sc_h2(e0, e1);
        }
        sum = fmaf(s0 + s1, exact_pow2(-(int)ps[q].y), sum);
        const int ch = pch + 2 * q;
        *reinterpret_cast<uint4*>(prow + ((ch ^ sw) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        *reinterpret_cast<uint4*>(prow + (((ch + 1) ^ sw) << 4)) = make_uint4(w[4], w[5], w[6], w[7]);
      }
      l = l * alpha + sum;
      m = m_new;
      fence_proxy_async();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready);
    }
    float l_other = 0.f;
    if (ok && n_kv > 0) ok = exchange(l, l_other);
    l += l_other;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (ok && n_kv > 0 && mbar_wait(pv_done, (n_kv - 1) & 1, abort_flag, p.status, 0xA32)) {
      tc_fence_after();
      __nv_bfloat16* orow = p.out + (long long)(q_row0 + tok) * p.ldo + head * D + ocol0;
#pragma unroll
      for (int c = 0; c < HO / 32; ++c) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(tO + t_lane + ocol0 + c * 32, r);
        tmem_ld_wait();
        if (row_live) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint4 o;
            o.x = pack_bf16x2(__uint_as_float(r[q * 8 + 0]) * inv, __uint_as_float(r[q * 8 + 1]) * inv);
            o.y = pack_bf16x2(__uint_as_float(r[q * 8 + 2]) * inv, __uint_as_float(r[q * 8 + 3]) * inv);
            o.z = pack_bf16x2(__uint_as_float(r[q * 8 + 4]) * inv, __uint_as_float(r[q * 8 + 5]) * inv);
            o.w = pack_bf16x2(__uint_as_float(r[q * 8 + 6]) * inv, __uint_as_float(r[q * 8 + 7]) * inv);
            *reinterpret_cast<uint4*>(orow + c * 32 + q * 8) = o;
          }
        }
      }
      if (p.ml && row_live && half == 0) p.ml[(long long)(q_row0 + tok) * p.Hq + head] = make_float2(m == -INFINITY ? 0.f : m, inv);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// ---------------------------------------------------------------------------------------------------------------- weights
constexpr int kSwThreads = 320;        // producer, issuer, eight warps that add
constexpr int kSwStages = 2;           // query tiles in shared memory, score buffers in TMEM

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
  static constexpr int kSmem = (1 + kSwStages) * kQ + kSwStages * kScRows * 8 + kScRows * 4 + 512 + 1024;
};

template <int D>
__global__ void __launch_bounds__(kSwThreads, 1)
scaled_chunk_weigh_kernel(const __grid_constant__ CUtensorMap tmap_q, const ScWeighParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int kQ = SwTile<D>::kQ;
  uint8_t* sK = smem;                                              // D / 64 sub-tiles [128 tokens][64 channels], bf16
  uint8_t* sQ = sK + kQ;                                           // kSwStages x the same of query rows
  float2* sMl = reinterpret_cast<float2*>(sQ + kSwStages * kQ);    // [stages][128] (M, 1 / l) of a row
  float* sSum = reinterpret_cast<float*>(sMl + kSwStages * kScRows);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sSum + kScRows);
  uint64_t* q_full = bars;                                         // [stages] one arrival + the tile's bytes
  uint64_t* q_empty = q_full + kSwStages;                          // [stages] QK done
  uint64_t* s_full = q_empty + kSwStages;                          // [stages]
  uint64_t* s_free = s_full + kSwStages;                           // [stages] 8 warps
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_free + kSwStages);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.G, toks = kScRows / G;
  const int b = p.tile_seq[blockIdx.x], k0 = p.tile_k0[blockIdx.x], kvh = blockIdx.y;
  const int L = min(p.seq_lens[b], p.bt_cols * kScPg);
  const int q_row0 = p.query_start_loc[b], q_len = p.query_start_loc[b + 1] - q_row0;
  const int ctx0 = L - q_len;
  // rows that see some of the tokens [k0, k0 + 128): positions [k0, k0 + 127 + window)
  const int r_lo = max(k0 - ctx0, 0) / toks * toks;
  const int r_hi = p.window > 0 ? min(q_len, k0 + kScRows - 1 + p.window - ctx0) : q_len;
  const int n_q = r_hi > r_lo ? (r_hi - r_lo + toks - 1) / toks : 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kSwStages; ++s) { mbar_init(&q_full[s], 1); mbar_init(&q_empty[s], 1); mbar_init(&s_full[s], 1); mbar_init(&s_free[s], 8); }
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
  __syncthreads();
  tc_fence_after();
  const uint32_t tS = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------------ producer: query rows, their M and 1 / l
    bool ok = true;
    for (int j = 0; j < n_q && ok; ++j) {
      const int s = j % kSwStages, q0 = r_lo + j * toks;
      if (lane == 0) ok = mbar_wait(&q_empty[s], ((j / kSwStages) & 1) ^ 1u, abort_flag, p.status, 0xB00) &&
                          mbar_wait(&s_free[s], ((j / kSwStages) & 1) ^ 1u, abort_flag, p.status, 0xB01);
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      if (!ok) break;
#pragma unroll
      for (int i = 0; i < kScRows; i += 32) {
        const int r = i + lane, tok = q0 + r / G;
        float2 x = make_float2(INFINITY, 0.f);                     // a row that is not there adds 2^-inf * 0
        if (r < toks * G && tok < q_len) x = p.ml[(long long)(q_row0 + tok) * p.Hq + kvh * G + r % G];
        sMl[s * kScRows + r] = x;
      }
      __syncwarp();
      if (lane == 0) {
        mbar_expect_tx(&q_full[s], (uint32_t)(D / 64) * 128u * (uint32_t)(toks * G));
#pragma unroll
        for (int c = 0; c < D / 64; ++c) tma_load_3d(sQ + s * kQ + c * kScSub, &tmap_q, &q_full[s], c * 64, kvh * G, q_row0 + q0);
      }
    }
    if (!ok)
      for (int i = 0; i < 64; ++i) __nanosleep(1000);
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer: S^T = K Q^T
    if (lane == 0) {
      constexpr uint32_t kIdesc = make_idesc(kScRows, kScRows, 1u);      // bf16 x bf16 -> f32
      const uint32_t aK = smem_u32(sK), aQ = smem_u32(sQ);
      for (int j = 0; j < n_q; ++j) {
        const int s = j % kSwStages;
        if (!mbar_wait(&q_full[s], (j / kSwStages) & 1, abort_flag, p.status, 0xB10)) break;
        tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint64_t ad = make_smem_desc_sw128(aK + (ks >> 2) * kScSub) + 2 * (ks & 3);
          const uint64_t bd = make_smem_desc_sw128(aQ + s * kQ + (ks >> 2) * kScSub) + 2 * (ks & 3);
          umma_f16(tS + s * kScRows, ad, bd, kIdesc, ks > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[s]);
        umma_commit(&q_empty[s]);
      }
    }
  } else {
    // ------------------------------------------------------------------ two threads a token, 64 rows each
    const int lane_group = warp & 3, half = (warp - 2) >> 2;
    const int trow = lane_group * 32 + lane, tok = k0 + trow;
    const uint32_t t_lane = (uint32_t)(lane_group * 32) << 16;
    float f = 0.f;
    if (tok < L) {
      const int blk = p.block_tables[(long long)b * p.bt_ld + tok / kScPg];
      if (blk >= 0 && blk < p.num_pages) f = p.scale_log2 * p.k_scale[blk * p.ks_ld + kvh * p.ks_h];
    }
    float total = 0.f;
    bool ok = true;
    for (int j = 0; j < n_q && ok; ++j) {
      const int s = j % kSwStages, q0 = r_lo + j * toks;
      ok = mbar_wait(&s_full[s], (j / kSwStages) & 1, abort_flag, p.status, 0xB20);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      tc_fence_after();
      uint32_t r[2][32];
#pragma unroll
      for (int c = 0; c < 2; ++c) tmem_ld_32x32b_x32(tS + s * kScRows + t_lane + half * 64 + c * 32, r[c]);
      tmem_ld_wait();
      const float4* ml = reinterpret_cast<const float4*>(sMl + s * kScRows + half * 64);
      // row r of the tile stands at position first + r / G: seen by tokens in (position - window, position]
      const int first = ctx0 + q0;
      const int there = min(toks, q_len - q0);             // rows behind them are another sequence's
      const bool all_seen = there == toks && k0 + kScRows - 1 <= first && (p.window == 0 || first + toks - 1 - p.window < k0);
      float a[4] = {0.f, 0.f, 0.f, 0.f};
      if (all_seen) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float4 x = ml[c * 16 + i / 2];
            a[i & 3] = fmaf(fast_exp2(fmaf(__uint_as_float(r[c][i]), f, -x.x)), x.y, a[i & 3]);
            a[(i & 3) + 1] = fmaf(fast_exp2(fmaf(__uint_as_float(r[c][i + 1]), f, -x.z)), x.w, a[(i & 3) + 1]);
          }
      } else {
        // columns of tokens [lo, hi) of the chunk see this lane's token
        const int c_lo = max(tok - first, 0) * G, c_hi = (p.window > 0 ? min(tok + p.window - first, there) : there) * G;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float4 x = ml[c * 16 + i / 2];
            const int col = half * 64 + c * 32 + i;
            const float e0 = fast_exp2(fmaf(__uint_as_float(r[c][i]), f, -x.x)) * x.y;
            const float e1 = fast_exp2(fmaf(__uint_as_float(r[c][i + 1]), f, -x.z)) * x.w;
            a[i & 3] += col >= c_lo && col < c_hi ? e0 : 0.f;
            a[(i & 3) + 1] += col + 1 >= c_lo && col + 1 < c_hi ? e1 : 0.f;
          }
      }
      total += (a[0] + a[1]) + (a[2] + a[3]);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_free[s]);
    }
    if (half == 1) sSum[trow] = total;
    asm volatile("bar.sync 1, 256;\n" ::: "memory");
    if (half == 0 && ok && tok < L && tok < p.width) p.weights[b * p.w_ld_b + kvh * p.w_ld_h + tok] += total + sSum[trow];
  }
  tc_fence_before();
  __syncthreads();
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

template <typename Kern, typename P>
int launch_tiles(Kern kern, int smem, dim3 grid, int threads, const CUtensorMap& tq, const P& p, cudaStream_t st) {
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem) != cudaSuccess) return -20;
  kern<<<grid, threads, smem, st>>>(tq, p);
  return cudaGetLastError() == cudaSuccess ? 0 : -20;
}

}  // namespace

// Rows of chunk sequences: `tiles` query tiles of 128 / G tokens, each (sequence, first token of the tile in its chunk); `ml` (or null) gets
// every row's reference and 1 / l.  With `weights`, tiles of 128 cached tokens follow, each (sequence, first token), whose sums grow by the
// rows' softmax weights.  Arguments as one record (see kv_scaled.cu).  -1: sizes or alignment outside of what the kernels take.
struct ChunkRecord {
  const void* q; long long ldq; void* out; long long ldo; const void* k_cache; const void* v_cache;
  const float* ks; long long ks_ld, ks_h; const float* vs; long long vs_ld, vs_h;
  const int* tables; long long bt_ld, bt_cols; const int* seq_lens; const int* starts;
  const int* tile_seq; const int* tile_q0; long long tiles, total_tokens, Hq, Hkv, D, window, num_pages; float* ml;
  const int* key_seq; const int* key_k0; long long key_tiles; float* weights; long long w_ld_b, w_ld_h, width; double scale; void* status;
  void* stream;
};
extern "C" int atlas_attn_scaled_chunk(const void* record) {
  const ChunkRecord& r = *static_cast<const ChunkRecord*>(record);
  const int D = (int)r.D;
  if (r.tiles <= 0) return 0;
  if ((D != 64 && D != 128 && D != 256) || r.Hkv <= 0 || r.Hkv > 65535 || r.Hq % r.Hkv || r.Hq / r.Hkv > kScRows) return -1;
  if ((reinterpret_cast<uintptr_t>(r.q) & 15) || r.ldq % 8 || r.ldo % 8 || (reinterpret_cast<uintptr_t>(r.out) & 15)) return -1;
  if ((reinterpret_cast<uintptr_t>(r.k_cache) | reinterpret_cast<uintptr_t>(r.v_cache)) & 15) return -1;
  if (r.bt_cols > (1 << 26) || r.tiles > 0x7fffffffll || r.total_tokens > 0x7fffffffll || (r.weights && !r.ml)) return -1;
  const int Hq = (int)r.Hq, Hkv = (int)r.Hkv, G = Hq / Hkv;
  CUtensorMap tq;
  if (int rc = query_map(&tq, r.q, r.ldq, (int)r.total_tokens, Hq, G, D)) return rc;
  const float scale_log2 = (float)(r.scale * 1.4426950408889634);
  status_t* status = (status_t*)r.status;
  cudaStream_t st = (cudaStream_t)r.stream;
  ScChunkParams p{(__nv_bfloat16*)r.out, r.ldo, (const uint8_t*)r.k_cache, (const uint8_t*)r.v_cache, r.ks, r.vs, r.ks_ld, r.vs_ld, (int)r.ks_h,
                  (int)r.vs_h, r.tables, (int)r.bt_ld, (int)r.bt_cols, r.seq_lens, r.starts, r.tile_seq, r.tile_q0, scale_log2, Hq, Hkv, G,
                  (int)r.window, (int)r.num_pages, reinterpret_cast<float2*>(r.ml), status};
  const dim3 grid((unsigned)r.tiles, Hkv);
  int rc;
  if (D == 64) rc = launch_tiles(scaled_chunk_kernel<64>, ScTile<64>::kSmem, grid, kScThreads, tq, p, st);
  else if (D == 128) rc = launch_tiles(scaled_chunk_kernel<128>, ScTile<128>::kSmem, grid, kScThreads, tq, p, st);
  else rc = launch_tiles(scaled_chunk_kernel<256>, ScTile<256>::kSmem, grid, kScThreads, tq, p, st);
  if (rc || !r.weights || r.key_tiles <= 0) return rc;
  ScWeighParams w{(const uint8_t*)r.k_cache, r.ks, r.ks_ld, (int)r.ks_h, r.tables, (int)r.bt_ld, (int)r.bt_cols, r.seq_lens, r.starts, r.key_seq,
                  r.key_k0, scale_log2, Hq, Hkv, G, (int)r.window, (int)r.num_pages, reinterpret_cast<const float2*>(r.ml), r.weights, r.w_ld_b,
                  r.w_ld_h, (int)r.width, status};
  const dim3 keys((unsigned)r.key_tiles, Hkv);
  if (D == 64) return launch_tiles(scaled_chunk_weigh_kernel<64>, SwTile<64>::kSmem, keys, kSwThreads, tq, w, st);
  if (D == 128) return launch_tiles(scaled_chunk_weigh_kernel<128>, SwTile<128>::kSmem, keys, kSwThreads, tq, w, st);
  return launch_tiles(scaled_chunk_weigh_kernel<256>, SwTile<256>::kSmem, keys, kSwThreads, tq, w, st);
}

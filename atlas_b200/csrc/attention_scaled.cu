// Single-token attention over the FP8 cache with a power-of-two scale per (page of 16 tokens, head), see kv_scaled.cu.
//
// With K^ and V^ the cache's numbers, s_j = a q . k^_j the score in the exp2 domain (a = softmax scale * log2(e) * the key page's scale) and
// 2^ev the value page's scale:
//
//   o = sum_j 2^(s_j) 2^ev v^_j / sum_j 2^(s_j) = sum_j p_j v^_j / sum_j p_j 2^-ev,     p_j = 2^(s_j + ev - M)
//
// so both scales ride in the exponent's multiply-add and the codes go to the tensor cores as they are.  M follows the maximum of s_j + ev, that is
// of what a token can add to the output, over the pages whose ev lie close together, and p is f16; pages whose ev is far from theirs have p as two
// bf16 terms and hardly move M (kv_scaled.cuh).  q is brought to 2^14 by a power of two; the sums are fp32.
//
// scaled_decode_kernel: bound by the cache's bytes (2 D a token and key head).  The pages of all (sequence, key head) pairs form one list, cut
// into equal runs, a run per warp: ragged batches and single long sequences fill the GPU alike.  A warp is on its own: it copies its pages
// into its ring of shared memory (cp.async.bulk, a page of K and one of V per slot), reads them as mma.sync fragments (tokens along M for
// the scores, channels along M for the outputs, heads along N) and leaves (M, l, O) of every pair it touched.  A piece's number is pair +
// warp, which no two pieces share.
// scaled_join_kernel and scaled_merge_kernel join the pieces of a pair.  scaled_weigh_kernel adds 2^(s - M) / l over the pair's heads to the running sums.
#include "common.cuh"
#include "host_api.h"
#include "kv_scaled.cuh"
#include "tc_util.cuh"

namespace atlas {

constexpr int kSdPage = 16;
constexpr int kSdRings = 192 * 1024;      // bytes of pages in flight per SM
// Warps of a block: sixteen where 128 registers a thread are enough for the output numbers (a page costs a warp 300 instructions, and with two
// warps a scheduler half of its time was waiting: 128 x 1152 tokens of 8 heads of 128 took 77 us), eight for wider heads or groups.
template <int D, int NT>
constexpr int kSdWarps = D * NT <= 128 ? 16 : 8;
constexpr int kSdLeast = 2;               // pages that make a run worth a warp of its own

struct ScaledDecodeParams {
  const __nv_bfloat16* q; long long ldq;
  __nv_bfloat16* out; long long ldo;
  const uint8_t* k_cache; const uint8_t* v_cache;
  const float* k_scale; const float* v_scale; long long ks_ld, vs_ld; int ks_h, vs_h;
  const int* block_tables; int bt_ld, bt_cols;
  const int* seq_lens; const int* query_start_loc;
  int nd, Hkv, G, tiles;                  // tiles: groups of at most 8 * NT query heads of a key head
  int window, num_pages;
  int warps;                              // of the whole grid
  float scale_log2;
  float* part_o; float* part_ml;          // piece: [D][cols], [cols] x (M, l)
  int cols;
  float* scores; long long width; int score_cols;      // [nd * Hkv][width][score_cols] or null
  float* ml;                              // [nd][Hq] x (M, 1 / l) or null
  status_t* status;
};

ATLAS_DEVICE void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
ATLAS_DEVICE void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
ATLAS_DEVICE uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
}

// Pages that the newest token of a sequence of `len` sees, and the first of them.
ATLAS_DEVICE int seen_pages(int len, int window, int& first) {
  const int lo = window > 0 ? max(len - window, 0) : 0;
  first = lo / kSdPage;
  return len > 0 ? (len + kSdPage - 1) / kSdPage - first : 0;
}
ATLAS_DEVICE int decode_len(const ScaledDecodeParams& p, int b) { return min(max(p.seq_lens[b], 0), p.bt_cols * kSdPage); }

// Pages of all sequences and of those before sequence `b`, the whole warp; up to 128 sequences in one round of loads.
ATLAS_DEVICE void count_pages(const ScaledDecodeParams& p, int b, int lane, int& all, int& before) {
  int sum = 0, pre = 0, first;
  for (int c = 0; c < p.nd; c += 128) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = c + 4 * lane + k;
      const int n = i < p.nd ? seen_pages(decode_len(p, i), p.window, first) : 0;
      sum += n;
      pre += i < b ? n : 0;
    }
  }
  all = __reduce_add_sync(0xffffffffu, sum);
  before = __reduce_add_sync(0xffffffffu, pre);
}
ATLAS_DEVICE int run_length(int pages, int warps) { return max((pages + warps - 1) / warps, kSdLeast); }

// One entry of the page list.
struct PageRef {
  int item;            // (sequence * Hkv + key head) * tiles + tile
  int tok0;            // first token of the page, one more for a far page (kv_scaled.cuh)
  int block;           // -1: an entry outside of the pool, skipped
  float sk, ev;        // key scale, value exponent
};

template <int D, int NT>
__global__ void __launch_bounds__(kSdWarps<D, NT> * 32, 1)
scaled_decode_kernel(const ScaledDecodeParams p) {
  constexpr int kWarps = kSdWarps<D, NT>, kSdRing = kSdRings / kWarps;
  constexpr int kPageBytes = kSdPage * D;
  constexpr int kStages = kSdRing / (2 * kPageBytes);
  constexpr int KS = D / 16;                      // k steps of a score
  constexpr int QB = D / 4;                       // channels of a lane's share of a row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[kWarps][kStages];
  __shared__ uint32_t abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * kSdRing;
  volatile uint32_t* abort_flag = &abort_word;
  if (threadIdx.x == 0) abort_word = 0;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&bars[warp][s], 1);
    mbar_fence_init();
  }
  __syncthreads();
  chain_trigger();
  chain_wait();
  const int w = warp * gridDim.x + blockIdx.x;    // neighbours in the list on different SMs
  const int hn = p.Hkv * p.tiles;
  int seen[4];                                    // pages of the first 128 sequences, four neighbours a lane: one round of loads
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    int first;
    const int b = 4 * lane + k;
    seen[k] = b < p.nd ? seen_pages(decode_len(p, b), p.window, first) : 0;
  }
  const int mine4 = seen[0] + seen[1] + seen[2] + seen[3];
  int incl = mine4;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  const int some = __shfl_sync(0xffffffffu, incl, 31);          // of those 128
  int all = some, before;
  if (p.nd > 128) count_pages(p, 0, lane, all, before);
  all *= hn;
  const int run = run_length(all, p.warps);
  const long long lo64 = (long long)w * run;
  if (lo64 >= all) return;
  const int n0 = (int)lo64, n1 = min(n0 + run, all);
  const int n = n1 - n0;

  // the sequence that entry n0 belongs to, and the entries before it
  int b0 = 0, base0 = 0;
  if (n0 < some * hn) {
    const int l = __ffs(__ballot_sync(0xffffffffu, incl * hn > n0)) - 1;
    int at = incl - mine4, b = 4 * lane;
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (b == 4 * lane + k && (at + seen[k]) * hn <= n0) { at += seen[k]; ++b; }
    b0 = __shfl_sync(0xffffffffu, b, l);
    base0 = __shfl_sync(0xffffffffu, at, l) * hn;
  } else {
    base0 = some * hn;
    for (int c = 128; c < p.nd; c += 32) {
      int first;
      const int mine = c + lane < p.nd ? seen_pages(decode_len(p, c + lane), p.window, first) * hn : 0;
      int in = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += x;
      }
      const unsigned past = __ballot_sync(0xffffffffu, base0 + in > n0);
      if (past) {
        const int l = __ffs(past) - 1;
        b0 = c + l;
        base0 += __shfl_sync(0xffffffffu, in - mine, l);
        break;
      }
      base0 += __shfl_sync(0xffffffffu, in, 31);
    }
  }
  // entries n0 + 32 c + lane
  auto fetch = [&](int c) -> PageRef {
    PageRef r{-1, 0, -1, 0.f, 0.f};
    const int i = 32 * c + lane;
    if (i >= n) return r;
    int at = n0 + i - base0, b = b0, first, np;
    for (;; ++b) {
      if (b >= p.nd) return r;
      np = seen_pages(decode_len(p, b), p.window, first);
      if (at < np * hn) break;
      at -= np * hn;
    }
    const int pair = at / np, pg = first + at % np;
    r.item = b * hn + pair;
    r.tok0 = pg * kSdPage;
    const int* row = p.block_tables + (long long)b * p.bt_ld;
    const int block = row[pg], ends[2] = {row[first], row[first + np - 1]};
    if (block >= 0 && block < p.num_pages) {
      const int h = pair / p.tiles;
      auto value_exponent = [&](int blk) { return scale_exponent(p.v_scale[blk * p.vs_ld + h * p.vs_h]); };
      const int ev = value_exponent(block);
      r.block = block;
      r.sk = p.k_scale[block * p.ks_ld + h * p.ks_h];
      r.ev = (float)ev;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (exponents_apart(ev, value_exponent((unsigned)ends[i] < (unsigned)p.num_pages ? ends[i] : block))) r.tok0 |= 1;
    }
    return r;
  };
  PageRef cur = fetch(0), nxt = fetch(1);
  int cur_chunk = 0;
  auto issue = [&](int i) {                         // entry i of this run into its slot; chunk cur_chunk or the next one
    const PageRef& r = (i >> 5) == cur_chunk ? cur : nxt;
    const int block = __shfl_sync(0xffffffffu, r.block, i & 31);
    const int item = __shfl_sync(0xffffffffu, r.item, i & 31);
    if (lane == 0) {
      const int s = i % kStages;
      uint64_t* bar = &bars[warp][s];
      uint8_t* dst = ring + s * 2 * kPageBytes;
      if (block >= 0) {
        const int h = (item / p.tiles) % p.Hkv;
        const long long at = ((long long)block * p.Hkv + h) * kPageBytes;
        mbar_expect_tx(bar, 2 * kPageBytes);
        bulk_page(dst, p.k_cache + at, kPageBytes, bar);
        bulk_page(dst + kPageBytes, p.v_cache + at, kPageBytes, bar);
      } else {
        mbar_arrive(bar);
      }
    }
  };
  for (int i = 0; i < min(n, kStages); ++i) issue(i);

  uint32_t qf[NT][KS][2];                           // queries as B fragments: head g of n-tile, channels t * QB + 4 step + 0 .. 3
  float a0[NT], a1[NT];                             // score factors of heads 2t, 2t + 1
  float m0[NT], m1[NT], l0[NT], l1[NT];
  float acc[NT][KS][4];                             // channels 16 i + g, + 8; heads 2t, 2t + 1
  int item = -1, len = 0, lo_tok = 0;

  auto flush = [&]() {
    const long long piece = (long long)item + w;
    float* o = p.part_o + piece * D * p.cols;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int c = nt * 8 + 2 * t;
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        l0[nt] += __shfl_xor_sync(0xffffffffu, l0[nt], x);
        l1[nt] += __shfl_xor_sync(0xffffffffu, l1[nt], x);
      }
      if (c < p.cols) {
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          *reinterpret_cast<float2*>(o + (16 * i + g) * p.cols + c) = make_float2(acc[nt][i][0], acc[nt][i][1]);
          *reinterpret_cast<float2*>(o + (16 * i + g + 8) * p.cols + c) = make_float2(acc[nt][i][2], acc[nt][i][3]);
        }
        if (g == 0) *reinterpret_cast<float4*>(p.part_ml + (piece * p.cols + c) * 2) = make_float4(m0[nt], l0[nt], m1[nt], l1[nt]);
      }
    }
  };
  auto begin = [&](int it) {
    item = it;
    const int tile = it % p.tiles, h = (it / p.tiles) % p.Hkv, b = it / hn;
    len = decode_len(p, b);
    lo_tok = p.window > 0 ? max(len - p.window, 0) : 0;
    const __nv_bfloat16* row = p.q + (long long)p.query_start_loc[b] * p.ldq;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int hg = tile * 8 * NT + nt * 8 + g;    // head of the group
      uint32_t raw[QB / 2];
#pragma unroll
      for (int i = 0; i < QB / 8; ++i) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (hg < p.G) v = *reinterpret_cast<const uint4*>(row + (h * p.G + hg) * D + t * QB + i * 8);
        raw[4 * i] = v.x; raw[4 * i + 1] = v.y; raw[4 * i + 2] = v.z; raw[4 * i + 3] = v.w;
      }
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < QB / 2; ++i) {
        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[i]));
        amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // largest magnitude to [2^13, 2^14): bf16 numbers are exact in f16 then down to 2^-30 of it, and off by 2^-38 of it at most below
      const int e = min(max(13 - ((int)(__float_as_uint(amax) >> 23) - 127), -114), 126);      // both powers are normal fp32 numbers
      const float up = __uint_as_float((uint32_t)(e + 127) << 23), down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[2 * i + j]));
          qf[nt][i][j] = pack_f16x2(f.x * up, f.y * up);
        }
      const float a = p.scale_log2 * down;
      a0[nt] = __shfl_sync(0xffffffffu, a, 8 * t);            // head 2t is the row g = 2t, lanes 8t ..
      a1[nt] = __shfl_sync(0xffffffffu, a, 8 * t + 4);
      m0[nt] = m1[nt] = -INFINITY;
      l0[nt] = l1[nt] = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[nt][i][j] = 0.f;
    }
  };

  const int tok_r = 4 * (g >> 1) + (g & 1);         // token of score row g; row g + 8 holds token tok_r + 2
  bool ok = true;
  for (int i = 0; i < n; ++i) {
    if ((i >> 5) != cur_chunk) {
      cur = nxt;
      ++cur_chunk;
      nxt = fetch(cur_chunk + 1);
    }
    const int it = __shfl_sync(0xffffffffu, cur.item, i & 31), tok0_far = __shfl_sync(0xffffffffu, cur.tok0, i & 31);
    const int tok0 = tok0_far & ~1;
    const bool far = tok0_far & 1;
    const int block = __shfl_sync(0xffffffffu, cur.block, i & 31);
    const float sk = __shfl_sync(0xffffffffu, cur.sk, i & 31), ev = __shfl_sync(0xffffffffu, cur.ev, i & 31);
    if (it != item) {
      if (item >= 0) flush();
      begin(it);
    }
    const int s = i % kStages;
    ok = mbar_wait(&bars[warp][s], (i / kStages) & 1, abort_flag, p.status, 0x900);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) break;
    if (block >= 0) {
      const uint8_t* kp = ring + s * 2 * kPageBytes;
      const uint8_t* vp = kp + kPageBytes;
      // ---- scores: rows g, g + 8 are tokens tok_r, tok_r + 2; a lane takes QB neighbouring channels of each
      float sc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[nt][j] = 0.f;
      const uint8_t* kr = kp + tok_r * D + t * QB;
#pragma unroll
      for (int c0 = 0; c0 < QB / 16; ++c0) {
        const uint4 x = *reinterpret_cast<const uint4*>(kr + c0 * 16), y = *reinterpret_cast<const uint4*>(kr + 2 * D + c0 * 16);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t f0 = e4m3x2_to_f16x2(xs[k] & 0xffffu), f1 = e4m3x2_to_f16x2(ys[k] & 0xffffu);
          const uint32_t f2 = e4m3x2_to_f16x2(xs[k] >> 16), f3 = e4m3x2_to_f16x2(ys[k] >> 16);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16(sc[nt], f0, f1, f2, f3, qf[nt][c0 * 4 + k][0], qf[nt][c0 * 4 + k][1]);
        }
      }
      // ---- softmax weights
      const bool whole = tok0 >= lo_tok && tok0 + kSdPage <= len;
      const bool see0 = whole || (tok0 + tok_r >= lo_tok && tok0 + tok_r < len);
      const bool see1 = whole || (tok0 + tok_r + 2 >= lo_tok && tok0 + tok_r + 2 < len);
      uint32_t vmask = 0xffffffffu;
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int tok = tok0 + 4 * t + j;
          if (tok < lo_tok || tok >= len) vmask &= ~(0xffu << (8 * j));
        }
      }
      uint32_t pb[NT][2], pl[NT][2];                  // p of tokens tok_r and tok_r + 2; a far page: the first terms, the second ones
      const float undo = __uint_as_float((uint32_t)(127 - (int)ev) << 23);     // 2^-ev
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float f0 = a0[nt] * sk, f1 = a1[nt] * sk;
        if (p.scores) {
          const int c = (it % p.tiles) * 8 * NT + nt * 8 + 2 * t;
          if (c < p.score_cols) {
            float* to = p.scores + ((long long)(it / p.tiles) * p.width + tok0 + tok_r) * p.score_cols + c;
            if (see0 && tok0 + tok_r < p.width) *reinterpret_cast<float2*>(to) = make_float2(sc[nt][0] * f0, sc[nt][1] * f1);
            if (see1 && tok0 + tok_r + 2 < p.width) *reinterpret_cast<float2*>(to + 2 * p.score_cols) = make_float2(sc[nt][2] * f0, sc[nt][3] * f1);
          }
        }
        const float s00 = see0 ? fmaf(sc[nt][0], f0, ev) : -INFINITY, s01 = see0 ? fmaf(sc[nt][1], f1, ev) : -INFINITY;
        const float s10 = see1 ? fmaf(sc[nt][2], f0, ev) : -INFINITY, s11 = see1 ? fmaf(sc[nt][3], f1, ev) : -INFINITY;
        const float slack = far ? kFarSlack : 0.f;
        float x0 = fmaxf(s00, s10) - slack, x1 = fmaxf(s01, s11) - slack;
        // The reference moves only when a score passes what set it by 2^8 (p stays inside f16): rarely after the first pages.
        if (__any_sync(0xffffffffu, x0 > m0[nt] + kMoves || x1 > m1[nt] + kMoves)) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, o));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, o));
          }
          const float n0m = fmaxf(m0[nt], x0 - kHeadroom), n1m = fmaxf(m1[nt], x1 - kHeadroom);
          const float r0 = m0[nt] == -INFINITY ? 0.f : fast_exp2(m0[nt] - n0m), r1 = m1[nt] == -INFINITY ? 0.f : fast_exp2(m1[nt] - n1m);
          m0[nt] = n0m; m1[nt] = n1m;
          l0[nt] *= r0; l1[nt] *= r1;
#pragma unroll
          for (int k = 0; k < KS; ++k) { acc[nt][k][0] *= r0; acc[nt][k][1] *= r1; acc[nt][k][2] *= r0; acc[nt][k][3] *= r1; }
        }
        const float r0 = m0[nt] == -INFINITY ? 0.f : m0[nt], r1 = m1[nt] == -INFINITY ? 0.f : m1[nt];
        const float p00 = fast_exp2(s00 - r0), p01 = fast_exp2(s01 - r1), p10 = fast_exp2(s10 - r0), p11 = fast_exp2(s11 - r1);
        l0[nt] += (p00 + p10) * undo;
        l1[nt] += (p01 + p11) * undo;
        if (!far) {
          pb[nt][0] = transpose8x8(pack_f16x2(p00, p01));
          pb[nt][1] = transpose8x8(pack_f16x2(p10, p11));
        } else {
          uint32_t hi[2], lo[2];
          two_terms(p00, p01, hi[0], lo[0]);
          two_terms(p10, p11, hi[1], lo[1]);
#pragma unroll
          for (int j = 0; j < 2; ++j) { pb[nt][j] = transpose8x8(hi[j]); pl[nt][j] = transpose8x8(lo[j]); }
        }
      }
      // ---- outputs: rows are channels, a lane takes tokens 4t .. 4t + 3 of channels 16 k + g and + 8
      auto values = [&](int k, uint32_t (&f)[4]) {
        const uint32_t x = *reinterpret_cast<const uint32_t*>(vp + (16 * k + g) * kSdPage + 4 * t) & vmask;
        const uint32_t y = *reinterpret_cast<const uint32_t*>(vp + (16 * k + g + 8) * kSdPage + 4 * t) & vmask;
        f[0] = e4m3x2_to_f16x2(x & 0xffffu); f[1] = e4m3x2_to_f16x2(y & 0xffffu);
        f[2] = e4m3x2_to_f16x2(x >> 16); f[3] = e4m3x2_to_f16x2(y >> 16);
      };
      if (!far) {
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t f[4];
          values(k, f);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16(acc[nt][k], f[0], f[1], f[2], f[3], pb[nt][0], pb[nt][1]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t f[4];
          values(k, f);
#pragma unroll
          for (int j = 0; j < 4; ++j) f[j] = h2_to_bf2(f[j]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_bf16(acc[nt][k], f[0], f[1], f[2], f[3], pb[nt][0], pb[nt][1]);
            mma_bf16(acc[nt][k], f[0], f[1], f[2], f[3], pl[nt][0], pl[nt][1]);
          }
        }
      }
    } else if (p.scores) {                            // a page outside of the pool is skipped, its tokens get no weight
      const int c0 = (it % p.tiles) * 8 * NT;
      for (int j = lane; j < kSdPage * 8 * NT; j += 32) {
        const int tok = tok0 + j / (8 * NT), c = c0 + j % (8 * NT);
        if (tok < len && tok < p.width && c < p.score_cols)
          p.scores[((long long)(it / p.tiles) * p.width + tok) * p.score_cols + c] = -INFINITY;
      }
    }
    __syncwarp();
    if (i + kStages < n) {
      fence_proxy_async();                          // this slot's reads before the copy that refills it
      issue(i + kStages);
    }
  }
  if (ok) flush();
  else
    for (int i = 0; i < 64; ++i) __nanosleep(1000);       // copies in flight land before the shared memory goes
}

// Pieces of a pair: warps [first page / run, last page / run] of the list; piece = pair + warp.
struct Pieces {
  long long first; int n;
};
ATLAS_DEVICE Pieces pieces_of(const ScaledDecodeParams& p, int item, int lane) {
  const int hn = p.Hkv * p.tiles, b = item / hn;
  int all, before, first;
  count_pages(p, b, lane, all, before);
  const int np = seen_pages(decode_len(p, b), p.window, first);
  const int run = run_length(all * hn, p.warps), start = before * hn + item % hn * np, w0 = start / run;
  return Pieces{(long long)item + w0, np > 0 ? (start + np - 1) / run - w0 + 1 : 0};
}

// Four neighbouring output numbers of a pair and their heads' references and sums, over pieces of it.
struct Joined {
  float m[4], l[4], o[4];
  ATLAS_DEVICE void clear() {
#pragma unroll
    for (int j = 0; j < 4; ++j) { m[j] = -INFINITY; l[j] = 0.f; o[j] = 0.f; }
  }
  // kAtOnce pieces, `step` apart, those before n: all their loads are in flight together
  template <int kAtOnce>
  ATLAS_DEVICE void add(const float2* ml, const float* part, const int (&c)[4], int cols, long long piece, int i, int step, int n) {
    float2 y[kAtOnce][4];
    float4 x[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int j = 0; j < 4; ++j) y[k][j] = make_float2(-INFINITY, 0.f);
      if (i + k * step < n) {
        x[k] = *reinterpret_cast<const float4*>(part + (i + k * step) * piece);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[k][j] = ml[(i + k * step) * cols + c[j]];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float top = m[j];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) top = fmaxf(top, y[k][j].x);
      const float ref = top == -INFINITY ? 0.f : top, f0 = fast_exp2(m[j] - ref);
      l[j] *= f0;
      o[j] *= f0;
      m[j] = top;
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const float f = fast_exp2(y[k][j].x - ref);        // a piece without a visible token: 2^-inf
        l[j] = fmaf(y[k][j].y, f, l[j]);
        o[j] = fmaf(j == 0 ? x[k].x : j == 1 ? x[k].y : j == 2 ? x[k].z : x[k].w, f, o[j]);
      }
    }
  }
};
ATLAS_DEVICE void store_joined(const ScaledDecodeParams& p, int b, int pair, int c, int d, int D, float m, float l, float o) {
  const int head = pair % p.tiles * p.cols + c, h = pair / p.tiles;
  if (head >= p.G) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;              // no token: zeros
  p.out[(long long)p.query_start_loc[b] * p.ldo + ((long long)h * p.G + head) * D + d] = __float2bfloat16_rn(o * inv);
  if (p.ml && d == 0) reinterpret_cast<float2*>(p.ml)[((long long)b * p.Hkv + h) * p.G + head] = make_float2(m == -INFINITY ? 0.f : m, inv);
}

// A few pieces a pair: a thread joins four neighbouring output numbers by itself, without a barrier.
template <int D>
__global__ void __launch_bounds__(128)
scaled_join_kernel(const ScaledDecodeParams p) {
  chain_trigger();
  chain_wait();
  const int item = blockIdx.x, hn = p.Hkv * p.tiles, b = item / hn, pair = item % hn;
  const Pieces pc = pieces_of(p, item, threadIdx.x & 31);
  const int e0 = 4 * (blockIdx.y * 128 + threadIdx.x);
  if (e0 >= D * p.cols) return;
  int c[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) c[j] = (e0 + j) % p.cols;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + pc.first * p.cols;
  const float* part = p.part_o + pc.first * D * p.cols + e0;
  Joined t;
  t.clear();
#pragma unroll 1
  for (int i = 0; i < pc.n; i += 4) t.add<4>(ml, part, c, p.cols, (long long)D * p.cols, i, 1, pc.n);
#pragma unroll
  for (int j = 0; j < 4; ++j) store_joined(p, b, pair, c[j], (e0 + j) / p.cols, D, t.m[j], t.l[j], t.o[j]);
}

// Many pieces a pair (long sequences, few pairs): sixteen warps take every sixteenth piece of the same 128 output numbers.
constexpr int kSdMergeWarps = 16;

template <int D>
__global__ void __launch_bounds__(kSdMergeWarps * 32)
scaled_merge_kernel(const ScaledDecodeParams p) {
  __shared__ float sm[kSdMergeWarps][128], sl[kSdMergeWarps][128], so[kSdMergeWarps][128];
  chain_trigger();
  chain_wait();
  const int item = blockIdx.x, hn = p.Hkv * p.tiles, b = item / hn, pair = item % hn;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Pieces pc = pieces_of(p, item, lane);
  const int e0 = blockIdx.y * 128 + 4 * lane;
  Joined t;
  t.clear();
  if (e0 < D * p.cols) {
    int c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = (e0 + j) % p.cols;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + pc.first * p.cols;
    const float* part = p.part_o + pc.first * D * p.cols + e0;
#pragma unroll 1
    for (int i = warp; i < pc.n; i += 4 * kSdMergeWarps) t.add<4>(ml, part, c, p.cols, (long long)D * p.cols, i, kSdMergeWarps, pc.n);
  }
  *reinterpret_cast<float4*>(&sm[warp][4 * lane]) = make_float4(t.m[0], t.m[1], t.m[2], t.m[3]);
  *reinterpret_cast<float4*>(&sl[warp][4 * lane]) = make_float4(t.l[0], t.l[1], t.l[2], t.l[3]);
  *reinterpret_cast<float4*>(&so[warp][4 * lane]) = make_float4(t.o[0], t.o[1], t.o[2], t.o[3]);
  __syncthreads();
  const int e = blockIdx.y * 128 + threadIdx.x;
  if (threadIdx.x >= 128 || e >= D * p.cols) return;
  float m = -INFINITY, l = 0.f, o = 0.f;
#pragma unroll
  for (int w = 0; w < kSdMergeWarps; ++w) m = fmaxf(m, sm[w][threadIdx.x]);
  const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int w = 0; w < kSdMergeWarps; ++w) {
    const float f = fast_exp2(sm[w][threadIdx.x] - ref);
    l = fmaf(sl[w][threadIdx.x], f, l);
    o = fmaf(so[w][threadIdx.x], f, o);
  }
  store_joined(p, b, pair, e % p.cols, e / p.cols, D, m, l, o);
}

// weights[b, h, j] += sum over the pair's heads of 2^(s - M) / l, a thread per token.
__global__ void __launch_bounds__(256)
scaled_weigh_kernel(const ScaledDecodeParams p, float* weights, long long w_ld_b, long long w_ld_h) {
  extern __shared__ float2 sh_ml[];
  chain_trigger();
  chain_wait();
  const int pair = blockIdx.x, b = pair / p.Hkv, h = pair % p.Hkv;
  const int len = decode_len(p, b), lo = p.window > 0 ? max(len - p.window, 0) : 0, end = (int)min((long long)len, p.width);
  for (int g = threadIdx.x; g < p.G; g += 256) sh_ml[g] = reinterpret_cast<const float2*>(p.ml)[(long long)b * p.Hkv * p.G + h * p.G + g];
  __syncthreads();
  for (int j = lo + blockIdx.y * 256 + threadIdx.x; j < end; j += gridDim.y * 256) {
    const float2* s = reinterpret_cast<const float2*>(p.scores + ((long long)pair * p.width + j) * p.score_cols);
    float sum = 0.f;
    for (int g = 0; g < p.G; g += 2) {
      const float2 x = s[g >> 1];
      sum += fast_exp2(x.x - sh_ml[g].x) * sh_ml[g].y;
      if (g + 1 < p.G) sum += fast_exp2(x.y - sh_ml[g + 1].x) * sh_ml[g + 1].y;
    }
    weights[b * w_ld_b + h * w_ld_h + j] += sum;
  }
}

}  // namespace atlas

using namespace atlas;

namespace {

template <int D, int NT>
int decode_launch(ScaledDecodeParams p, int blocks, int items, long long max_len, cudaStream_t st) {
  constexpr int smem = kSdRings;
  p.warps = blocks * kSdWarps<D, NT>;
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(scaled_decode_kernel<D, NT>), smem) != cudaSuccess) return -20;
  if (launch_chain(scaled_decode_kernel<D, NT>, dim3(blocks), dim3(kSdWarps<D, NT> * 32), smem, st, p) != cudaSuccess) { cudaGetLastError(); return -20; }
  // Single threads join up to four pieces a pair on average (128 x 1152 tokens of 8 heads, 3 a pair: 65 us with the attention, 89 by blocks), and
  // up to sixteen if no pair can have hundreds (a warp has two pages or more, and its share of the longest sequence's list): 32 x 4096 ragged
  // tokens with weights, 9 a pair, 59 us, 62 by blocks; but 3 x 65531 tokens, 197 a pair, 89 us, 42 by blocks.  Both come to the same sums; a
  // captured step chooses by the length that it was captured for.
  const long long most = min((max_len + 2 * kSdPage - 1) / (2 * kSdPage), (long long)p.warps * p.nd / items + 1) + 1;
  const bool few = 4ll * items >= p.warps || (16ll * items >= p.warps && most <= 256);
  const cudaError_t e = few ? launch_chain(scaled_join_kernel<D>, dim3(items, (D * p.cols + 511) / 512), dim3(128), 0, st, p)
                            : launch_chain(scaled_merge_kernel<D>, dim3(items, (D * p.cols + 127) / 128), dim3(kSdMergeWarps * 32), 0, st, p);
  if (e != cudaSuccess) { cudaGetLastError(); return -20; }
  return 0;
}

}  // namespace

// Decode rows of a step: sequence b's row is query_start_loc[b].  Arguments as one record (see kv_scaled.cu).  Workspaces: part_o [pieces][D]
// [cols] and part_ml [pieces][cols][2] with cols = min(G rounded up to two, 16) and pieces = pairs + 16 blocks, a pair being (sequence, key head,
// group of 16 query heads).  With `weights`: scores [nd * Hkv][width][G rounded up to two], ml [nd][Hq][2] and the sums
// [sequence][head][token], at least `width` tokens each, of which no sequence has more.  -1: sizes or alignment outside of what the kernels take.
struct DecodeRecord {
  const void* q; long long ldq; void* out; long long ldo; const void* k_cache; const void* v_cache;
  const float* ks; long long ks_ld, ks_h; const float* vs; long long vs_ld, vs_h;
  const int* tables; long long bt_ld, bt_cols; const int* seq_lens; const int* starts;
  long long nd, Hq, Hkv, D, window, num_pages, max_len, blocks; float* part_o; float* part_ml;
  float* scores; long long width; float* ml; float* weights; long long w_ld_b, w_ld_h; double scale; void* status; void* stream;
};
extern "C" int atlas_attn_scaled_decode(const void* record) {
  const DecodeRecord& r = *static_cast<const DecodeRecord*>(record);
  const int D = (int)r.D;
  if (r.nd <= 0) return 0;
  if ((D != 64 && D != 128 && D != 256) || r.Hkv <= 0 || r.Hq < r.Hkv || r.Hq % r.Hkv || r.Hq / r.Hkv > 128 || r.ldq % 8 || (reinterpret_cast<uintptr_t>(r.q) & 15)) return -1;
  if ((reinterpret_cast<uintptr_t>(r.k_cache) | reinterpret_cast<uintptr_t>(r.v_cache)) & 15) return -1;
  if (!(r.scale >= 0x1p-60 && r.scale <= 0x1p60)) return -1;
  ScaledDecodeParams p;
  p.q = (const __nv_bfloat16*)r.q; p.ldq = r.ldq; p.out = (__nv_bfloat16*)r.out; p.ldo = r.ldo;
  p.k_cache = (const uint8_t*)r.k_cache; p.v_cache = (const uint8_t*)r.v_cache;
  p.k_scale = r.ks; p.v_scale = r.vs; p.ks_ld = r.ks_ld; p.vs_ld = r.vs_ld; p.ks_h = (int)r.ks_h; p.vs_h = (int)r.vs_h;
  p.block_tables = r.tables; p.bt_ld = (int)r.bt_ld; p.bt_cols = (int)r.bt_cols; p.seq_lens = r.seq_lens; p.query_start_loc = r.starts;
  p.nd = (int)r.nd; p.Hkv = (int)r.Hkv; p.G = (int)(r.Hq / r.Hkv); p.tiles = (p.G + 15) / 16;
  p.cols = p.G <= 16 ? (p.G + 1) / 2 * 2 : 16;
  // the list's entries and the runs' bounds are 32-bit numbers
  const long long items = r.nd * r.Hkv * p.tiles;
  if (items * r.bt_cols > 0x3fffffffll || items > 0x7fffffffll || r.bt_cols > (1 << 25) || r.window < 0 || r.window > (1 << 29) || r.blocks <= 0 || r.blocks > 65535) return -1;
  p.window = (int)r.window; p.num_pages = (int)r.num_pages;
  p.scale_log2 = (float)(r.scale * 1.4426950408889634);
  p.part_o = r.part_o; p.part_ml = r.part_ml;
  p.scores = r.weights ? r.scores : nullptr; p.width = r.width; p.score_cols = (p.G + 1) / 2 * 2; p.ml = r.weights ? r.ml : nullptr;
  p.status = (status_t*)r.status;
  cudaStream_t st = (cudaStream_t)r.stream;
  const int blocks = (int)r.blocks, n = (int)items;
  int rc;
  if (p.G <= 8) rc = D == 64 ? decode_launch<64, 1>(p, blocks, n, r.max_len, st) : D == 128 ? decode_launch<128, 1>(p, blocks, n, r.max_len, st) : decode_launch<256, 1>(p, blocks, n, r.max_len, st);
  else rc = D == 64 ? decode_launch<64, 2>(p, blocks, n, r.max_len, st) : D == 128 ? decode_launch<128, 2>(p, blocks, n, r.max_len, st) : decode_launch<256, 2>(p, blocks, n, r.max_len, st);
  if (rc || !r.weights) return rc;
  const long long chunks = (r.max_len + 1023) / 1024;
  if (launch_chain(scaled_weigh_kernel, dim3((unsigned)(r.nd * r.Hkv), (unsigned)(chunks < 1 ? 1 : chunks < 64 ? chunks : 64)), dim3(256),
                   (size_t)p.G * sizeof(float2), st, p, r.weights, r.w_ld_b, r.w_ld_h) != cudaSuccess) { cudaGetLastError(); return -20; }
  return 0;
}

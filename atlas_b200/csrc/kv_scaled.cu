// The FP8 cache whose scales go by block: one power of two for the 16 tokens of a page of one head, keys and values apart.
//
//   scale(page, head) = 2^e, the smallest e in [-60, 60] with max |x| <= 448 * 2^e;   code = e4m3(x / 2^e)
//
// A power of two makes every rescaling exact except where a code falls below e4m3's normal range: appending to a page may raise its scale
// (it never lowers it), and the codes already there are then multiplied by 2^(e_old - e).  A page whose first token is written starts anew.
// It also lets the attention kernels fold the scales into exponents.
//
//   kv_scaled_write_kernel   head norm + rotation + scales + rounding + paged write, rotated queries beside it
//   kv_scaled_read_kernel    the cache's values as rows (bf16: an e4m3 number times a power of two is one exactly)
//   kv_evict_select_kernel   per sequence and head: the heaviest tokens' positions, in order
//   kv_evict_move_kernel     those tokens into new pages, rescaled
//
// Layout as in elementwise.cu: K [pages, Hkv, 16, D], V [pages, Hkv, D, 16].  All four are bound by memory: a warp owns the 16 tokens of
// one page and head, a lane D / 32 neighbouring channels of every token, so that K rows, V rows (16 bytes) and bf16 rows are all moved in
// whole sectors without a transposition.
#include "common.cuh"
#include "host_api.h"

namespace atlas {

constexpr int kScPage = 16;
constexpr int kScLow = -60, kScHigh = 60;

// Smallest e with a <= 448 * 2^e = 1.75 * 2^(e + 8): the exponent field, one more if the mantissa is above 1.75's.
ATLAS_DEVICE int block_exponent(float a) {
  const int e = (int)((__float_as_uint(a) + 0x1FFFFFu) >> 23) - 127 - 8;
  return min(max(e, kScLow), kScHigh);
}
ATLAS_DEVICE float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }       // e in [-126, 127]
ATLAS_DEVICE int exponent_of(float s) { return (int)((__float_as_uint(s) >> 23) & 255u) - 127; }

template <int V>
struct Codes { uint32_t w[(V + 3) / 4]; };            // V consecutive e4m3 codes, V in {2, 4, 8}

template <int V>
ATLAS_DEVICE Codes<V> load_codes(const uint8_t* p) {
  Codes<V> c;
  if constexpr (V == 2) c.w[0] = *reinterpret_cast<const uint16_t*>(p);
  else if constexpr (V == 4) c.w[0] = *reinterpret_cast<const uint32_t*>(p);
  else { const uint2 t = *reinterpret_cast<const uint2*>(p); c.w[0] = t.x; c.w[1] = t.y; }
  return c;
}
template <int V>
ATLAS_DEVICE void store_codes(uint8_t* p, const Codes<V>& c) {
  if constexpr (V == 2) *reinterpret_cast<uint16_t*>(p) = (uint16_t)c.w[0];
  else if constexpr (V == 4) *reinterpret_cast<uint32_t*>(p) = c.w[0];
  else *reinterpret_cast<uint2*>(p) = make_uint2(c.w[0], c.w[1]);
}
ATLAS_DEVICE float2 codes2_to_f32(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(h) : "h"((uint16_t)two));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}
ATLAS_DEVICE uint32_t f32_to_codes2(float a, float b) { return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3); }
template <int V>
ATLAS_DEVICE void widen(const Codes<V>& c, float (&f)[V]) {
#pragma unroll
  for (int i = 0; i < V; i += 2) {
    const float2 t = codes2_to_f32((c.w[i >> 2] >> (8 * (i & 3))) & 0xFFFFu);
    f[i] = t.x; f[i + 1] = t.y;
  }
}
template <int V>
ATLAS_DEVICE Codes<V> narrow(const float (&f)[V], float by) {
  Codes<V> c;
#pragma unroll
  for (int w = 0; w < (V + 3) / 4; ++w) c.w[w] = 0;
#pragma unroll
  for (int i = 0; i < V; i += 2) c.w[i >> 2] |= f32_to_codes2(f[i] * by, f[i + 1] * by) << (8 * (i & 3));
  return c;
}
// sixteen codes (one channel of a page's values) times a power of two
ATLAS_DEVICE uint4 rescale16(uint4 v, float by) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = codes2_to_f32(w[i] & 0xFFFFu), b = codes2_to_f32(w[i] >> 16);
    w[i] = f32_to_codes2(a.x * by, a.y * by) | (f32_to_codes2(b.x * by, b.y * by) << 16);
  }
  return v;
}
template <int V>
ATLAS_DEVICE void load_row(const __nv_bfloat16* p, float (&f)[V]) {
  uint32_t w[V / 2];
  if constexpr (V == 2) w[0] = *reinterpret_cast<const uint32_t*>(p);
  else if constexpr (V == 4) { const uint2 t = *reinterpret_cast<const uint2*>(p); w[0] = t.x; w[1] = t.y; }
  else { const uint4 t = *reinterpret_cast<const uint4*>(p); w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w; }
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const float2 t = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
    f[2 * i] = t.x; f[2 * i + 1] = t.y;
  }
}
template <int V>
ATLAS_DEVICE void store_row(__nv_bfloat16* p, const float (&f)[V]) {
  uint32_t w[V / 2];
#pragma unroll
  for (int i = 0; i < V / 2; ++i) w[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
  if constexpr (V == 2) *reinterpret_cast<uint32_t*>(p) = w[0];
  else if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

struct ScaledWriteParams {
  const __nv_bfloat16* q; long long ldq;
  __nv_bfloat16* q_out; long long ldqo;
  const __nv_bfloat16* k; long long ldk;
  const __nv_bfloat16* v; long long ldv;
  const int* positions; const float* rope;      // rope: [positions, rotary]: cos half, sin half
  const __nv_bfloat16* q_norm; const __nv_bfloat16* k_norm;
  uint8_t* k_cache; uint8_t* v_cache;
  float* k_scale; float* v_scale; long long ks_ld, vs_ld; int ks_h, vs_h;      // scale of (page, head) at [page * ld + head * h]
  const int* slots;
  int T, Hq, Hkv, rotary, num_pages, plus_one, norm_dim;
  int rows_per_block, kv_blocks_x, kv_blocks_y;  // blocks [0, kv_blocks_x * kv_blocks_y) write the cache, the others turn queries
  float eps;
};

// Head norm and rotation of one head, `V` neighbouring channels a lane, in fp32 throughout.  The rotation's partner channel, half the
// rotary width away, belongs to a lane `hl` further on or back.
template <int V>
struct Turn {
  float c[V], s[V];      // of this lane's channels; the partner's share comes with its sign
  int hl;                // lanes between partners; lanes from 2 * hl on are not rotated
  ATLAS_DEVICE void angles(const float* rope_row, int rotary, int lane) {
    hl = rotary / (2 * V);
    if (lane >= 2 * hl) return;
    const int d = (lane < hl ? lane : lane - hl) * V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      c[i] = __ldg(rope_row + d + i);
      const float t = __ldg(rope_row + rotary / 2 + d + i);
      s[i] = lane < hl ? -t : t;
    }
  }
  ATLAS_DEVICE void operator()(float (&x)[V], const float (&w)[V], bool normed, int norm_dim, float eps, int lane) const {
    if (normed) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) ss += x[i] * x[i];
      const float r = rsqrtf(warp_sum(ss) / (float)norm_dim + eps);
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] *= r * w[i];
    }
    if (hl == 0) return;
    const int from = lane < hl ? lane + hl : (lane < 2 * hl ? lane - hl : lane);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float y = __shfl_sync(0xffffffffu, x[i], from);
      if (lane < 2 * hl) x[i] = x[i] * c[i] + y * s[i];
    }
  }
};

template <int V>
ATLAS_DEVICE void norm_weights(const __nv_bfloat16* w, int plus_one, int lane, float (&out)[V]) {
  if (!w) return;
  load_row<V>(w + lane * V, out);
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] += plus_one ? 1.f : 0.f;
}

constexpr int kWriteHeads = 8;      // query heads of a token that one warp turns with the same angles

// Cache blocks: a warp takes the rows of one step that fall into one page, for one head's keys or values.  A run of such rows starts where
// the slot is not the one behind the row before.  Two passes over its rows (the second one hits L1): the largest magnitude, then codes.
template <int D>
__global__ void __launch_bounds__(256)
kv_scaled_write_kernel(const ScaledWriteParams p) {
  constexpr int V = D / 32;
  chain_trigger();
  chain_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kv_blocks = p.kv_blocks_x * p.kv_blocks_y;
  float w[V];
  Turn<V> turn;
  turn.hl = 0;
  if ((int)blockIdx.x >= kv_blocks) {
    const int groups = (p.Hq + kWriteHeads - 1) / kWriteHeads;
    const long long unit = (long long)(blockIdx.x - kv_blocks) * 8 + warp;
    if (unit >= (long long)p.T * groups) return;
    const int t = (int)(unit / groups), h0 = (int)(unit % groups) * kWriteHeads;
    if (p.rotary) turn.angles(p.rope + (long long)p.positions[t] * p.rotary, p.rotary, lane);
    norm_weights<V>(p.q_norm, p.plus_one, lane, w);
    float x[kWriteHeads][V];
#pragma unroll
    for (int i = 0; i < kWriteHeads; ++i)
      if (h0 + i < p.Hq) load_row<V>(p.q + t * p.ldq + (h0 + i) * D + lane * V, x[i]);
#pragma unroll
    for (int i = 0; i < kWriteHeads; ++i) {
      if (h0 + i >= p.Hq) return;
      turn(x[i], w, p.q_norm != nullptr, p.norm_dim, p.eps, lane);
      store_row<V>(p.q_out + t * p.ldqo + (h0 + i) * D + lane * V, x[i]);
    }
    return;
  }
  const int task = (blockIdx.x / p.kv_blocks_x) * 8 + warp;           // (K heads, then V heads)
  if (task >= 2 * p.Hkv) return;
  const bool is_k = task < p.Hkv;
  const int h = is_k ? task : task - p.Hkv;
  const __nv_bfloat16* src = (is_k ? p.k : p.v) + h * D + lane * V;
  const long long ld = is_k ? p.ldk : p.ldv;
  if (is_k) norm_weights<V>(p.k_norm, p.plus_one, lane, w);
  const bool normed = is_k && p.k_norm != nullptr;
  const int row0 = (blockIdx.x % p.kv_blocks_x) * p.rows_per_block;
  for (int t0 = row0; t0 < min(row0 + p.rows_per_block, p.T); ++t0) {
    const int slot = p.slots[t0];
    if (slot < 0 || slot >= p.num_pages * kScPage) continue;
    const int page = slot / kScPage, off = slot % kScPage;
    if (off > 0 && t0 > 0 && p.slots[t0 - 1] == slot - 1) continue;    // the row before began this run
    // rows t0 .. t0 + n - 1 fill slots off .. off + n - 1 of the page
    const bool mine = lane < kScPage - off && t0 + lane < p.T && p.slots[min(t0 + lane, p.T - 1)] == slot + lane;
    const int n = __ffs(~__ballot_sync(0xffffffffu, mine)) - 1;
    const long long base = ((long long)page * p.Hkv + h) * (kScPage * D);
    float* scale_at = is_k ? p.k_scale + page * p.ks_ld + h * p.ks_h : p.v_scale + page * p.vs_ld + h * p.vs_h;
    const float before = off > 0 ? *scale_at : 0.f;
    auto row = [&](int r, float (&x)[V]) {
      load_row<V>(src + (long long)(t0 + r) * ld, x);
      if (is_k) {
        if (p.rotary) turn.angles(p.rope + (long long)p.positions[t0 + r] * p.rotary, p.rotary, lane);
        turn(x, w, normed, p.norm_dim, p.eps, lane);
      }
    };
    float amax = 0.f;
#pragma unroll 4
    for (int r = 0; r < n; ++r) {
      float x[V];
      row(r, x);
#pragma unroll
      for (int i = 0; i < V; ++i) amax = fmaxf(amax, fabsf(x[i]));
    }
    amax = warp_max(amax);
    int e = block_exponent(amax);
    const int e_old = exponent_of(before);
    if (off > 0) e = max(e, e_old);
    const float inv = pow2i(-e);
    const bool raised = off > 0 && e != e_old;
    const float shift = raised ? pow2i(max(e_old - e, -126)) : 1.f;
    if (is_k) {
      uint8_t* page_k = p.k_cache + base + lane * V;
      if (raised)
        for (int r = 0; r < off; ++r) {
          float x[V];
          widen<V>(load_codes<V>(page_k + r * D), x);
          store_codes<V>(page_k + r * D, narrow<V>(x, shift));
        }
#pragma unroll 4
      for (int r = 0; r < n; ++r) {
        float x[V];
        row(r, x);
        store_codes<V>(page_k + (off + r) * D, narrow<V>(x, inv));
      }
    } else {
      uint4* page_v = reinterpret_cast<uint4*>(p.v_cache + base) + lane * V;       // [channel] 16 tokens
      uint32_t out[V][4];
      const bool whole = n == kScPage;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        uint4 was = make_uint4(0, 0, 0, 0);
        if (!whole) was = page_v[i];
        const uint4 moved = raised ? rescale16(was, shift) : was;
        const uint32_t* a = reinterpret_cast<const uint32_t*>(&was);
        const uint32_t* b = reinterpret_cast<const uint32_t*>(&moved);
#pragma unroll
        for (int j = 0; j < 4; ++j) {                                  // tokens before `off` moved, those behind the run as they were
          const int lo = min(max(off - 4 * j, 0), 4);
          const uint32_t m = lo == 4 ? 0xffffffffu : ((1u << (8 * lo)) - 1u);
          out[i][j] = (b[j] & m) | (a[j] & ~m);
        }
      }
#pragma unroll
      for (int tok = 0; tok < kScPage; ++tok) {
        if (tok < off || tok >= off + n) continue;                     // the same for all lanes
        float x[V];
        load_row<V>(src + (long long)(t0 + tok - off) * ld, x);
        const Codes<V> c = narrow<V>(x, inv);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const uint32_t code = (c.w[i >> 2] >> (8 * (i & 3))) & 0xFFu;
          out[i][tok >> 2] = (out[i][tok >> 2] & ~(0xFFu << (8 * (tok & 3)))) | (code << (8 * (tok & 3)));
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) page_v[i] = make_uint4(out[i][0], out[i][1], out[i][2], out[i][3]);
    }
    __syncwarp();
    if (lane == 0 && (off == 0 || raised)) *scale_at = pow2i(e);
  }
}

// ---------------------------------------------------------------------------------------------------------------- reading
struct ScaledCache {
  const uint8_t* k; const uint8_t* v;
  const float* ks; const float* vs; long long ks_ld, vs_ld; int ks_h, vs_h;
  int Hkv, num_pages;
};

template <int D>
__global__ void __launch_bounds__(256)
kv_scaled_read_kernel(const ScaledCache c, const int* __restrict__ tables, int bt_ld, int bt_cols, const int* __restrict__ lens, int max_len, int pages,
                      long long units, __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out) {
  constexpr int V = D / 32;
  chain_trigger();
  chain_wait();
  const int lane = threadIdx.x & 31;
  long long u = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (u >= units) return;
  const bool is_k = (u & 1) == 0;
  u >>= 1;
  const int h = (int)(u % c.Hkv);
  const long long bp = u / c.Hkv;
  const int b = (int)(bp / pages), pg = (int)(bp % pages);
  const int len = min(lens[b], min(max_len, bt_cols * kScPage));
  const int live = min(max(len - pg * kScPage, 0), kScPage), rows = min(max_len - pg * kScPage, kScPage);
  const long long step = (long long)c.Hkv * D;
  __nv_bfloat16* out = (is_k ? k_out : v_out) + (((long long)b * max_len + pg * kScPage) * c.Hkv + h) * D + lane * V;
  float zero[V];
#pragma unroll
  for (int i = 0; i < V; ++i) zero[i] = 0.f;
  int page = live > 0 ? tables[(long long)b * bt_ld + pg] : -1;
  const bool ok = page >= 0 && page < c.num_pages;
  if (!ok) {
    for (int r = 0; r < rows; ++r) store_row<V>(out + r * step, zero);
    return;
  }
  const float s = is_k ? c.ks[page * c.ks_ld + h * c.ks_h] : c.vs[page * c.vs_ld + h * c.vs_h];
  const uint8_t* base = (is_k ? c.k : c.v) + ((long long)page * c.Hkv + h) * (kScPage * D);
  if (is_k) {
    Codes<V> codes[kScPage];
#pragma unroll
    for (int r = 0; r < kScPage; ++r) codes[r] = load_codes<V>(base + r * D + lane * V);
#pragma unroll
    for (int r = 0; r < kScPage; ++r) {
      if (r >= rows) break;
      float x[V];
      widen<V>(codes[r], x);
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = r < live ? x[i] * s : 0.f;
      store_row<V>(out + r * step, x);
    }
  } else {
    uint4 col[V];
#pragma unroll
    for (int i = 0; i < V; ++i) col[i] = reinterpret_cast<const uint4*>(base)[lane * V + i];
#pragma unroll
    for (int r = 0; r < kScPage; r += 2) {
      float a[V], z[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const uint32_t word = reinterpret_cast<const uint32_t*>(&col[i])[r >> 2];
        const float2 t = codes2_to_f32((word >> (8 * (r & 3))) & 0xFFFFu);
        a[i] = r < live ? t.x * s : 0.f;
        z[i] = r + 1 < live ? t.y * s : 0.f;
      }
      if (r < rows) store_row<V>(out + r * step, a);
      if (r + 1 < rows) store_row<V>(out + (r + 1) * step, z);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------- evicting
// Weights in the order of unsigned numbers: NaN below everything, -0 with +0.
ATLAS_DEVICE uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct SelectParams {
  const float* weights; long long w_ld_b, w_ld_h;      // [sequence][head][token]
  const int* seq_lens;
  int* new_lens; int* kept; float* w_out;              // [B], [B, Hkv, keep], [B, Hkv, keep]
  int Hkv, keep, sink, recent, width;
};

constexpr int kSelThreads = 1024;
constexpr int kSelBins = 2048;

// One block per (sequence, head).  The `room`-th largest key among the tokens between sink and recent, 11, 11 and 10 bits at a time
// (a histogram each, weights come from L2), then the positions in order: every warp counts its span of tokens, the spans' counts are
// summed, and each warp writes its own.
__global__ void __launch_bounds__(kSelThreads)
kv_evict_select_kernel(const SelectParams p) {
  __shared__ uint32_t hist[kSelBins];
  __shared__ uint32_t warp_a[32], warp_b[32];
  __shared__ uint32_t sh_bin, sh_above;
  chain_trigger();
  chain_wait();
  const int b = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int len = min(max(p.seq_lens[b], 0), p.width);
  const int kept = min(len, p.keep);
  const float* w = p.weights + b * p.w_ld_b + h * p.w_ld_h;
  int* out = p.kept + ((long long)b * p.Hkv + h) * p.keep;
  float* wo = p.w_out + ((long long)b * p.Hkv + h) * p.keep;
  if (h == 0 && tid == 0) p.new_lens[b] = kept;
  for (int i = kept + tid; i < p.keep; i += kSelThreads) { out[i] = -1; wo[i] = 0.f; }
  if (len <= p.keep) {
    for (int i = tid; i < len; i += kSelThreads) { out[i] = i; wo[i] = w[i]; }
    return;
  }
  const int lo = p.sink, hi = len - p.recent;
  int room = p.keep - p.sink - p.recent;                // >= 0; hi - lo = len - sink - recent > room
  uint32_t prefix = 0, mask = 0;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < kSelBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int i0 = lo; i0 < hi; i0 += kSelThreads * 4) {
      uint32_t key[4];
      bool in[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * kSelThreads + tid;
        in[u] = i < hi;
        key[u] = in[u] ? weight_key(w[i]) : 0u;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bool hit = in[u] && (key[u] & mask) == prefix;
        const uint32_t bin = (key[u] >> shift) & ((1u << bits) - 1u);
        // tokens that nothing looked at share one bin: a warp adds equal neighbours at once
        const uint32_t first = __shfl_sync(0xffffffffu, bin, 0);
        const uint32_t same = __ballot_sync(0xffffffffu, hit && bin == first);
        if (hit && bin != first) atomicAdd(&hist[bin], 1u);
        if (lane == 0 && same) atomicAdd(&hist[first], (uint32_t)__popc(same));
      }
    }
    __syncthreads();
    // the bin that holds the room-th largest: suffix sums over 2048 bins, two a thread
    const uint32_t c0 = hist[2 * tid], c1 = hist[2 * tid + 1];
    uint32_t suffix = c0 + c1;                           // inclusive sum from this thread's bins to the warp's end
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t n = __shfl_down_sync(0xffffffffu, suffix, o);
      if (lane + o < 32) suffix += n;
    }
    if (lane == 0) warp_a[warp] = suffix;
    if (tid == 0) { sh_bin = 0; sh_above = 0; }
    __syncthreads();
    uint32_t above = suffix - c0 - c1;
    for (int i = warp + 1; i < 32; ++i) above += warp_a[i];
    // exactly one bin has above < room <= above + count (room >= 1)
    if (room > 0) {
      if (above < (uint32_t)room && (uint32_t)room <= above + c1) { sh_bin = 2 * tid + 1; sh_above = above; }
      else if (above + c1 < (uint32_t)room && (uint32_t)room <= above + c1 + c0) { sh_bin = 2 * tid; sh_above = above + c1; }
    }
    __syncthreads();
    prefix |= sh_bin << shift;
    mask |= ((1u << bits) - 1u) << shift;
    room -= (int)sh_above;
    __syncthreads();
  }
  // keys above `prefix` stay, the first `room` that equal it too
  if (p.keep - p.sink - p.recent == 0) { prefix = 0xffffffffu; room = 0; }
  for (int i = tid; i < p.sink; i += kSelThreads) { out[i] = i; wo[i] = w[i]; }
  for (int i = tid; i < p.recent; i += kSelThreads) { out[p.keep - p.recent + i] = hi + i; wo[p.keep - p.recent + i] = w[hi + i]; }
  const int span = ((hi - lo + 31) / 32 + 31) / 32 * 32;             // tokens of a warp
  const int s0 = lo + warp * span, s1 = min(s0 + span, hi);
  uint32_t more = 0, equal = 0;
#pragma unroll 4
  for (int i = s0 + lane; i < s1; i += 32) {
    const uint32_t key = weight_key(w[i]);
    more += key > prefix;
    equal += key == prefix;
  }
  more = (uint32_t)__reduce_add_sync(0xffffffffu, more);
  equal = (uint32_t)__reduce_add_sync(0xffffffffu, equal);
  if (lane == 0) { warp_a[warp] = more; warp_b[warp] = equal; }
  __syncthreads();
  int at = p.sink, ties = 0;
  for (int i = 0; i < warp; ++i) {
    at += (int)warp_a[i];
    ties += (int)warp_b[i];
  }
  at += min(ties, room);
#pragma unroll 4
  for (int i0 = s0; i0 < s1; i0 += 32) {
    const int i = i0 + lane;
    const float x = i < s1 ? w[i] : 0.f;
    const uint32_t key = weight_key(x);
    const bool eq = i < s1 && key == prefix;
    const uint32_t eqs = __ballot_sync(0xffffffffu, eq);
    const bool take = (i < s1 && key > prefix) || (eq && ties + __popc(eqs & ((1u << lane) - 1u)) < room);
    const uint32_t takes = __ballot_sync(0xffffffffu, take);
    const int to = at + __popc(takes & ((1u << lane) - 1u));
    if (take && to < p.keep - p.recent) { out[to] = i; wo[to] = x; }
    at += __popc(takes);
    ties += __popc(eqs);
  }
}

struct MoveParams {
  ScaledCache from;
  uint8_t* k; uint8_t* v; float* ks; float* vs;
  const int* tables; int bt_ld;
  const int* to; int to_ld;
  const int* kept; const int* new_lens;
  int keep, pages; long long units;
};

// A warp writes one page of one head.  A kept value token's 16-byte columns hold its neighbours too: every source page is read once as a
// whole for all tokens that come from it.
template <int D>
__global__ void __launch_bounds__(256)
kv_evict_move_kernel(const MoveParams p) {
  constexpr int V = D / 32;
  chain_trigger();
  chain_wait();
  const int lane = threadIdx.x & 31;
  long long u = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (u >= p.units) return;
  const bool is_k = (u & 1) == 0;
  u >>= 1;
  const ScaledCache& c = p.from;
  const int pg = (int)(u % p.pages);
  u /= p.pages;
  const int h = (int)(u % c.Hkv), b = (int)(u / c.Hkv);
  const int live = min(p.new_lens[b] - pg * kScPage, kScPage);
  if (live <= 0) return;
  const int dst = p.to[(long long)b * p.to_ld + pg];
  if (dst < 0 || dst >= c.num_pages) return;
  // lane r < 16: where token r of the new page comes from
  int page = -1, off = 0;
  float scale = 0.f;
  if (lane < live) {
    const int pos = p.kept[((long long)b * c.Hkv + h) * p.keep + pg * kScPage + lane];
    page = p.tables[(long long)b * p.bt_ld + pos / kScPage];
    off = pos % kScPage;
    if (page < 0 || page >= c.num_pages) page = -1;
    else scale = is_k ? c.ks[page * c.ks_ld + h * c.ks_h] : c.vs[page * c.vs_ld + h * c.vs_h];
  }
  const uint8_t* pool = (is_k ? c.k : c.v) + (long long)h * (kScPage * D);
  const long long step = (long long)c.Hkv * (kScPage * D);
  Codes<V> codes[kScPage];
#pragma unroll
  for (int r = 0; r < kScPage; ++r)
#pragma unroll
    for (int i = 0; i < (V + 3) / 4; ++i) codes[r].w[i] = 0;
  if (is_k) {
#pragma unroll
    for (int r = 0; r < kScPage; ++r) {
      const int pr = __shfl_sync(0xffffffffu, page, r), o = __shfl_sync(0xffffffffu, off, r);
      if (pr >= 0) codes[r] = load_codes<V>(pool + pr * step + o * D + lane * V);
    }
  } else {
    int have = -1;
    uint4 col[V];
#pragma unroll
    for (int r = 0; r < kScPage; ++r) {
      const int pr = __shfl_sync(0xffffffffu, page, r), o = __shfl_sync(0xffffffffu, off, r);
      if (pr < 0) continue;
      if (pr != have) {
        have = pr;
#pragma unroll
        for (int i = 0; i < V; ++i) col[i] = reinterpret_cast<const uint4*>(pool + pr * step)[lane * V + i];
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const uint32_t lo = (o & 4) ? col[i].y : col[i].x, hi = (o & 4) ? col[i].w : col[i].z;
        const uint32_t code = (((o & 8) ? hi : lo) >> (8 * (o & 3))) & 0xFFu;
        codes[r].w[i >> 2] |= code << (8 * (i & 3));
      }
    }
  }
  float amax = 0.f;
#pragma unroll
  for (int r = 0; r < kScPage; ++r) {
    const float s = __shfl_sync(0xffffffffu, scale, r);
    float x[V];
    widen<V>(codes[r], x);
#pragma unroll
    for (int i = 0; i < V; ++i) amax = fmaxf(amax, fabsf(x[i]) * s);
  }
  amax = warp_max(amax);
  const int e = block_exponent(amax);
#pragma unroll
  for (int r = 0; r < kScPage; ++r) {
    const float s = __shfl_sync(0xffffffffu, scale, r);
    float x[V];
    widen<V>(codes[r], x);
    codes[r] = narrow<V>(x, s * pow2i(-e));      // a power of two: exact
  }
  const long long base = ((long long)dst * c.Hkv + h) * (kScPage * D);
  if (is_k) {
#pragma unroll
    for (int r = 0; r < kScPage; ++r) store_codes<V>(p.k + base + r * D + lane * V, codes[r]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      uint32_t out[4] = {0, 0, 0, 0};
#pragma unroll
      for (int r = 0; r < kScPage; ++r) out[r >> 2] |= ((codes[r].w[i >> 2] >> (8 * (i & 3))) & 0xFFu) << (8 * (r & 3));
      reinterpret_cast<uint4*>(p.v + base)[lane * V + i] = make_uint4(out[0], out[1], out[2], out[3]);
    }
  }
  if (lane == 0) {
    if (is_k) p.ks[dst * c.ks_ld + h * c.ks_h] = pow2i(e);
    else p.vs[dst * c.vs_ld + h * c.vs_h] = pow2i(e);
  }
}

}  // namespace atlas

using namespace atlas;

namespace {

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <template <int> class F, typename... A>
int by_width(int D, A... a) {
  if (D == 64) return F<64>::launch(a...);
  if (D == 128) return F<128>::launch(a...);
  if (D == 256) return F<256>::launch(a...);
  return -1;
}

int launched(cudaError_t e) {
  if (e != cudaSuccess) { cudaGetLastError(); return -20; }
  return 0;
}

template <int D>
struct Write {
  static int launch(const ScaledWriteParams& p, unsigned blocks, cudaStream_t st) {
    return launched(launch_chain_if(p.T <= 256, kv_scaled_write_kernel<D>, dim3(blocks), dim3(256), 0, st, p));
  }
};
template <int D>
struct Read {
  static int launch(const ScaledCache& c, const int* tables, int bt_ld, int bt_cols, const int* lens, int max_len, int pages, long long units,
                    __nv_bfloat16* k, __nv_bfloat16* v, cudaStream_t st) {
    return launched(launch_chain(kv_scaled_read_kernel<D>, dim3((unsigned)((units + 7) / 8)), dim3(256), 0, st, c, tables, bt_ld, bt_cols, lens, max_len,
                                 pages, units, k, v));
  }
};
template <int D>
struct Move {
  static int launch(const MoveParams& p, cudaStream_t st) {
    return launched(launch_chain(kv_evict_move_kernel<D>, dim3((unsigned)((p.units + 7) / 8)), dim3(256), 0, st, p));
  }
};

}  // namespace

// -1: sizes or alignment that the kernels do not take (16-token pages, heads of 64, 128 or 256, rows on 2 * D / 32 elements, rotary widths
// of whole lanes); -20: a launch failed.
extern "C" int atlas_kv_scaled_write(const void* q, long long ldq, void* q_out, long long ldqo, const void* k, long long ldk, const void* v,
                                     long long ldv, const int* positions, const float* rope, const void* q_norm, const void* k_norm,
                                     void* k_cache, void* v_cache, float* k_scale, long long ks_ld, int ks_h, float* v_scale, long long vs_ld,
                                     int vs_h, const int* slots, int T, int Hq, int Hkv, int D, int rotary, int num_pages, int plus_one,
                                     int norm_dim, float eps, void* stream) {
  if (T <= 0) return 0;
  if (D != 64 && D != 128 && D != 256) return -1;
  const int V = D / 32;
  if (rotary < 0 || rotary > D || rotary % (2 * V) || num_pages <= 0 || num_pages > (1 << 27) || Hkv <= 0 || Hq < 0) return -1;
  if (ldq % V || ldqo % V || ldk % V || ldv % V || !aligned(k, 2 * V) || !aligned(v, 2 * V) || !aligned(k_cache, 16) || !aligned(v_cache, 16)) return -1;
  if (Hq > 0 && (!aligned(q, 2 * V) || !aligned(q_out, 2 * V))) return -1;
  if ((q_norm && !aligned(q_norm, 2 * V)) || (k_norm && !aligned(k_norm, 2 * V))) return -1;
  ScaledWriteParams p;
  p.q = (const __nv_bfloat16*)q; p.ldq = ldq; p.q_out = (__nv_bfloat16*)q_out; p.ldqo = ldqo;
  p.k = (const __nv_bfloat16*)k; p.ldk = ldk; p.v = (const __nv_bfloat16*)v; p.ldv = ldv;
  p.positions = positions; p.rope = rope; p.q_norm = (const __nv_bfloat16*)q_norm; p.k_norm = (const __nv_bfloat16*)k_norm;
  p.k_cache = (uint8_t*)k_cache; p.v_cache = (uint8_t*)v_cache;
  p.k_scale = k_scale; p.v_scale = v_scale; p.ks_ld = ks_ld; p.vs_ld = vs_ld; p.ks_h = ks_h; p.vs_h = vs_h;
  p.slots = slots; p.T = T; p.Hq = Hq; p.Hkv = Hkv; p.rotary = rotary; p.num_pages = num_pages; p.plus_one = plus_one;
  p.norm_dim = norm_dim > 0 ? norm_dim : D; p.eps = eps;
  // Decode steps: every row begins a run, one row a block.  Prompts: one row in 16 does, and blocks of four rows leave fewer blocks empty.
  p.rows_per_block = T <= 512 ? 1 : 4;
  p.kv_blocks_x = (T + p.rows_per_block - 1) / p.rows_per_block;
  p.kv_blocks_y = (2 * Hkv + 7) / 8;
  const long long q_units = (long long)T * ((Hq + kWriteHeads - 1) / kWriteHeads);
  const long long blocks = (long long)p.kv_blocks_x * p.kv_blocks_y + (q_units + 7) / 8;
  if (blocks > 0x7fffffffll) return -1;
  return by_width<Write>(D, p, (unsigned)blocks, (cudaStream_t)stream);
}

extern "C" int atlas_kv_scaled_read(const void* k_cache, const void* v_cache, const float* k_scale, long long ks_ld, int ks_h,
                                    const float* v_scale, long long vs_ld, int vs_h, const int* tables, int bt_ld, int bt_cols, const int* lens, int B,
                                    int max_len, int Hkv, int D, int num_pages, void* k_out, void* v_out, void* stream) {
  if (B <= 0 || max_len <= 0) return 0;
  if (bt_cols > (1 << 26)) return -1;
  if (!aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(k_out, 16) || !aligned(v_out, 16)) return -1;
  const ScaledCache c{(const uint8_t*)k_cache, (const uint8_t*)v_cache, k_scale, v_scale, ks_ld, vs_ld, ks_h, vs_h, Hkv, num_pages};
  const int pages = (max_len + kScPage - 1) / kScPage;
  const long long units = 2ll * B * pages * Hkv;
  if ((units + 7) / 8 > 0x7fffffffll) return -1;
  return by_width<Read>(D, c, tables, bt_ld, bt_cols, lens, max_len, pages, units, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, (cudaStream_t)stream);
}

extern "C" int atlas_kv_evict(void* k_cache, void* v_cache, float* k_scale, long long ks_ld, int ks_h, float* v_scale, long long vs_ld, int vs_h,
                              const int* tables, int bt_ld, const int* seq_lens, const float* weights, long long w_ld_b, long long w_ld_h, int width,
                              int B, int Hkv, int D, int num_pages, int keep, int sink, int recent, const int* to, int to_ld, int* new_lens,
                              int* kept, float* w_out, void* stream) {
  if (B <= 0) return 0;
  if (keep <= 0 || sink < 0 || recent < 0 || sink + recent > keep || !aligned(k_cache, 16) || !aligned(v_cache, 16)) return -1;
  if (D != 64 && D != 128 && D != 256) return -1;
  cudaStream_t st = (cudaStream_t)stream;
  SelectParams s{weights, w_ld_b, w_ld_h, seq_lens, new_lens, kept, w_out, Hkv, keep, sink, recent, width};
  const int rc = launched(launch_chain(kv_evict_select_kernel, dim3(B * Hkv), dim3(kSelThreads), 0, st, s));
  if (rc) return rc;
  MoveParams m;
  m.from = ScaledCache{(const uint8_t*)k_cache, (const uint8_t*)v_cache, k_scale, v_scale, ks_ld, vs_ld, ks_h, vs_h, Hkv, num_pages};
  m.k = (uint8_t*)k_cache; m.v = (uint8_t*)v_cache; m.ks = k_scale; m.vs = v_scale;
  m.tables = tables; m.bt_ld = bt_ld; m.to = to; m.to_ld = to_ld; m.kept = kept; m.new_lens = new_lens; m.keep = keep;
  m.pages = (keep + kScPage - 1) / kScPage;
  m.units = 2ll * B * Hkv * m.pages;
  return by_width<Move>(D, m, st);
}

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
// Layout as in elementwise.cu: K [pages, Hkv, 16, D], V [pages, Hkv, D, 16].  All four are bound by memory: warps own the tokens of one page
// and head, a lane D / 32 neighbouring channels of every token, so that K rows, V rows (16 bytes) and bf16 rows are all moved in whole
// sectors without a transposition.
#include "common.cuh"
#include "host_api.h"
#include "kv_scaled.cuh"

namespace atlas {

constexpr int kScPage = 16;
constexpr int kScLow = -60, kScHigh = 60;

// Smallest e with a <= 448 * 2^e = 1.75 * 2^(e + 8): the exponent field, one more if the mantissa is above 1.75's.
ATLAS_DEVICE int block_exponent(float a) {
  const int e = (int)((__float_as_uint(a) + 0x1FFFFFu) >> 23) - 127 - 8;
  return min(max(e, kScLow), kScHigh);
}

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
  const uint32_t h = e4m3x2_to_f16x2(two);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
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
template <int V>
struct Raw { uint32_t w[V / 2]; };                    // V consecutive bf16 numbers

template <int V>
ATLAS_DEVICE Raw<V> load_raw(const __nv_bfloat16* p) {
  Raw<V> r;
  if constexpr (V == 2) r.w[0] = *reinterpret_cast<const uint32_t*>(p);
  else if constexpr (V == 4) { const uint2 t = *reinterpret_cast<const uint2*>(p); r.w[0] = t.x; r.w[1] = t.y; }
  else { const uint4 t = *reinterpret_cast<const uint4*>(p); r.w[0] = t.x; r.w[1] = t.y; r.w[2] = t.z; r.w[3] = t.w; }
  return r;
}
template <int V>
ATLAS_DEVICE void unpack(const Raw<V>& r, float (&f)[V]) {
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const float2 t = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r.w[i]));
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
    if (lane >= 2 * hl) return;
    const float* at = rope_row + (lane < hl ? lane : lane - hl) * V;
    load_floats(at, c);
    load_floats(at + rotary / 2, s);
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = lane < hl ? -s[i] : s[i];
  }
  static ATLAS_DEVICE void load_floats(const float* at, float (&f)[V]) {      // rows of the table start on 16 bytes, or 8 for V = 2
    if constexpr (V == 2) {
      const float2 t = __ldg(reinterpret_cast<const float2*>(at));
      f[0] = t.x; f[1] = t.y;
    } else {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 t = __ldg(reinterpret_cast<const float4*>(at + i));
        f[i] = t.x; f[i + 1] = t.y; f[i + 2] = t.z; f[i + 3] = t.w;
      }
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
  unpack<V>(load_raw<V>(w + lane * V), out);
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] += plus_one ? 1.f : 0.f;
}

// Queries: 16 bytes a lane, so that D / 8 lanes hold a head and a warp 256 / D of them; four such loads of one token are in flight and share
// the angles.
template <int D>
ATLAS_DEVICE void turn_queries(const ScaledWriteParams& p, unsigned unit, int lane) {
  constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes, kHeads = 4 * kAtOnce;
  const unsigned groups = (unsigned)(p.Hq + kHeads - 1) / kHeads, t = unit / groups;
  if (t >= (unsigned)p.T) return;
  const int h0 = (int)(unit % groups) * kHeads + lane / kLanes, sl = lane % kLanes;
  const __nv_bfloat16* src = p.q + (long long)t * p.ldq + h0 * D + sl * 8;
  __nv_bfloat16* dst = p.q_out + (long long)t * p.ldqo + h0 * D + sl * 8;
  Raw<8> raw[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (h0 + j * kAtOnce < p.Hq) raw[j] = load_raw<8>(src + j * kAtOnce * D);
  const int hl = p.rotary / 16;                      // lanes between the channels of a rotated pair
  float c[8], s[8], w[8];
  if (sl < 2 * hl) {
    const float* at = p.rope + (long long)p.positions[t] * p.rotary + (sl < hl ? sl : sl - hl) * 8;
    Turn<8>::load_floats(at, c);
    Turn<8>::load_floats(at + p.rotary / 2, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = sl < hl ? -s[i] : s[i];
  }
  norm_weights<8>(p.q_norm, p.plus_one, sl, w);
  const int from = sl < hl ? lane + hl : (sl < 2 * hl ? lane - hl : lane);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float x[8];
    unpack<8>(raw[j], x);
    if (p.q_norm) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(ss / (float)p.norm_dim + p.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= r * w[i];
    }
    if (hl > 0)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = __shfl_sync(0xffffffffu, x[i], from);
        if (sl < 2 * hl) x[i] = x[i] * c[i] + y * s[i];
      }
    if (h0 + j * kAtOnce < p.Hq) store_row<8>(dst + j * kAtOnce * D, x);
  }
}

// Cache blocks: `W` warps take the rows of one step that fall into one page, for one head's keys and values, in groups of four slots; a run of
// such rows starts where the slot is not the one behind the row before.  Prompts: four warps, a group each, every row loaded and turned once
// and waiting in registers for the page's largest magnitude.  (A warp per page took 30 us for 517 rows of 256-wide heads, sixteen rows' angles
// one after the other; four take 9.)  Decode steps: one warp, since most runs are one row, and 128 rows of 8 heads fit the GPU at once (6 us; with
// four warps 11); a longer run is loaded and turned twice.
template <int D, int W>
__global__ void __launch_bounds__(256, D == 256 ? 2 : 4)
kv_scaled_write_kernel(const ScaledWriteParams p) {
  constexpr int V = D / 32;
  __shared__ float2 sh_amax[8];
  __shared__ uint32_t sh_v[W > 1 ? 8 / W : 1][W > 1 ? D * 4 : 1];      // value pages: [channel] 16 tokens
  chain_trigger();
  chain_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kv_blocks = p.kv_blocks_x * p.kv_blocks_y;
  if ((int)blockIdx.x >= kv_blocks) {
    turn_queries<D>(p, (blockIdx.x - kv_blocks) * 8 + warp, lane);
    return;
  }
  const int local = warp / W;
  const int h = (blockIdx.x / p.kv_blocks_x) * (8 / W) + local;
  const bool on = h < p.Hkv;
  if (W == 1 && !on) return;
  float w[V];
  Turn<V> turn;
  turn.hl = p.rotary / (2 * V);
  const __nv_bfloat16* k_src = p.k + h * D + lane * V;
  const __nv_bfloat16* v_src = p.v + h * D + lane * V;
  norm_weights<V>(p.k_norm, p.plus_one, lane, w);
  const bool normed = p.k_norm != nullptr;
  // the runs that start in this block's rows, all lanes looking at once
  const int row0 = (blockIdx.x % p.kv_blocks_x) * p.rows_per_block;
  bool starts = false;
  if (lane < p.rows_per_block && row0 + lane < p.T) {
    const int slot = p.slots[row0 + lane];
    starts = slot >= 0 && slot < p.num_pages * kScPage && !(slot % kScPage > 0 && row0 + lane > 0 && p.slots[row0 + lane - 1] == slot - 1);
  }
  uint32_t runs = __ballot_sync(0xffffffffu, starts);                  // the same for the whole block
  while (runs) {
    const int t0 = row0 + __ffs(runs) - 1;
    runs &= runs - 1;
    const int slot = p.slots[t0], page = slot / kScPage, off = slot % kScPage;
    // rows t0 .. t0 + n - 1 fill slots off .. off + n - 1 of the page
    const int mine_t = min(t0 + lane, p.T - 1);
    const bool mine = lane < kScPage - off && t0 + lane < p.T && p.slots[mine_t] == slot + lane;
    const int my_pos = p.rotary ? p.positions[mine_t] : 0;
    const int n = __ffs(~__ballot_sync(0xffffffffu, mine)) - 1;
    const long long base = ((long long)page * p.Hkv + h) * (kScPage * D);
    float* ks_at = p.k_scale + page * p.ks_ld + h * p.ks_h;
    float* vs_at = p.v_scale + page * p.vs_ld + h * p.vs_h;
    float k_before = 0.f, v_before = 0.f;
    if (on && off > 0) { k_before = *ks_at; v_before = *vs_at; }
    const int g_lo = W == 1 ? off / 4 : (warp & 3), g_hi = W == 1 ? (off + n - 1) / 4 : (warp & 3);      // groups with rows of the run
    float x[4][V];
    Raw<V> v_raw[4];
    auto load_group = [&](int g, float2 amax) {
      Raw<V> k_raw[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 4 * g + j - off;
        if (r >= 0 && r < n) {
          k_raw[j] = load_raw<V>(k_src + (long long)(t0 + r) * p.ldk);
          v_raw[j] = load_raw<V>(v_src + (long long)(t0 + r) * p.ldv);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 4 * g + j - off;
        if (r < 0 || r >= n) continue;
        float y[V];
        unpack<V>(v_raw[j], y);
#pragma unroll
        for (int i = 0; i < V; ++i) amax.y = fmaxf(amax.y, fabsf(y[i]));
        unpack<V>(k_raw[j], x[j]);
        if (p.rotary) turn.angles(p.rope + (long long)__shfl_sync(0xffffffffu, my_pos, r) * p.rotary, p.rotary, lane);
        turn(x[j], w, normed, p.norm_dim, p.eps, lane);
#pragma unroll
        for (int i = 0; i < V; ++i) amax.x = fmaxf(amax.x, fabsf(x[j][i]));
      }
      return amax;
    };
    float2 amax = make_float2(0.f, 0.f);
    if (on)
      for (int g = g_lo; g <= g_hi; ++g) amax = load_group(g, amax);
    amax.x = warp_max(amax.x);
    amax.y = warp_max(amax.y);
    if constexpr (W > 1) {
      if (lane == 0) sh_amax[warp] = amax;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float2 o = sh_amax[local * W + i];
        amax.x = fmaxf(amax.x, o.x);
        amax.y = fmaxf(amax.y, o.y);
      }
    }
    int ke = block_exponent(amax.x), ve = block_exponent(amax.y);
    const int ke_old = scale_exponent(k_before), ve_old = scale_exponent(v_before);
    if (off > 0) { ke = max(ke, ke_old); ve = max(ve, ve_old); }
    const bool k_raised = off > 0 && ke != ke_old, v_raised = off > 0 && ve != ve_old;
    const float k_shift = exact_pow2(max(ke_old - ke, -126)), v_shift = exact_pow2(max(ve_old - ve, -126));      // used where the scale rose
    // a group's tokens: rows of the run, tokens before them (to the new scale, if it rose), tokens behind them (as they were)
    auto store_group = [&](int g) {
      uint8_t* page_k = p.k_cache + base + lane * V;
      uint32_t word[V];                                                // four tokens of each channel: a word of the channel's sixteen
#pragma unroll
      for (int i = 0; i < V; ++i) word[i] = 0;
      uint32_t fresh = 0, old = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int s = 4 * g + j, r = s - off;
        if (r >= 0 && r < n) {
          store_codes<V>(page_k + s * D, narrow<V>(x[j], exact_pow2(-ke)));
          fresh |= 0xFFu << (8 * j);
          float y[V];
          unpack<V>(v_raw[j], y);
          const Codes<V> c = narrow<V>(y, exact_pow2(-ve));
#pragma unroll
          for (int i = 0; i < V; ++i) word[i] |= ((c.w[i >> 2] >> (8 * (i & 3))) & 0xFFu) << (8 * j);
        } else if (r < 0) {
          old |= 0xFFu << (8 * j);
          if (k_raised) {
            float y[V];
            widen<V>(load_codes<V>(page_k + s * D), y);
            store_codes<V>(page_k + s * D, narrow<V>(y, k_shift));
          }
        }
      }
      uint32_t* at = reinterpret_cast<uint32_t*>(p.v_cache + base) + lane * V * 4 + g;
      if (fresh != 0xffffffffu) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const uint32_t was = at[4 * i];
          uint32_t moved = was;
          if (v_raised && old) {
            const float2 lo = codes2_to_f32(was & 0xFFFFu), hi = codes2_to_f32(was >> 16);
            moved = f32_to_codes2(lo.x * v_shift, lo.y * v_shift) | (f32_to_codes2(hi.x * v_shift, hi.y * v_shift) << 16);
          }
          word[i] = (word[i] & fresh) | (moved & old) | (was & ~(fresh | old));
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if constexpr (W > 1) sh_v[local][(lane * V + i) * 4 + g] = word[i];
        else at[4 * i] = word[i];
      }
    };
    if constexpr (W == 1) {
      for (int g = k_raised || v_raised ? 0 : g_lo; g <= g_hi; ++g) {
        if (g >= g_lo && g_lo != g_hi) load_group(g, amax);
        store_group(g);
      }
      __syncwarp();
    } else {
      if (on) store_group(warp & 3);
      __syncthreads();
      if (on) {                                                        // whole channels, 16 bytes each
        uint4* page_v = reinterpret_cast<uint4*>(p.v_cache + base);
        for (int c = (warp & 3) * 32 + lane; c < D; c += 128) page_v[c] = reinterpret_cast<const uint4*>(sh_v[local])[c];
      }
    }
    if (on && lane == 0 && (W == 1 || (warp & 3) == 0)) {
      if (off == 0 || k_raised) *ks_at = exact_pow2(ke);
      if (off == 0 || v_raised) *vs_at = exact_pow2(ve);
    }
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
                      unsigned units, __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out) {
  constexpr int V = D / 32;
  chain_trigger();
  chain_wait();
  const int lane = threadIdx.x & 31;
  unsigned u = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (u >= units) return;
  const bool is_k = (u & 1) == 0;
  u >>= 1;
  const int h = (int)(u % (unsigned)c.Hkv);
  const unsigned bp = u / (unsigned)c.Hkv;
  const int b = (int)(bp / (unsigned)pages), pg = (int)(bp % (unsigned)pages);
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

ATLAS_DEVICE uint32_t ld_cluster_u32(const void* mine, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];\n" : "=r"(v) : "r"(cluster_map_shared(smem_u32(mine), rank)) : "memory");
  return v;
}
ATLAS_DEVICE uint2 ld_cluster_u32x2(const void* mine, uint32_t rank) {
  uint2 v;
  asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(cluster_map_shared(smem_u32(mine), rank)) : "memory");
  return v;
}
ATLAS_DEVICE void st_cluster_u32x2(void* mine, uint32_t rank, uint2 v) {
  asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};\n" ::"r"(cluster_map_shared(smem_u32(mine), rank)), "r"(v.x), "r"(v.y) : "memory");
}

// One block, or a cluster of up to eight, per (sequence, head); a warp has a span of neighbouring tokens.  The `room`-th largest key among the tokens
// between sink and recent, 11, 11 and 10 bits at a time: every block counts its tokens, then sums its share of the bins over the cluster's
// blocks and hands the sums to all of them through distributed shared memory, a load and a store of two bins a thread.  (Blocks that sum all
// bins for themselves read 64 KB from the others: 34 in place of 22 us for eight heads of 65531 tokens.)  Then the positions in order: the
// spans' counts are summed and each warp writes its own.  The first kHeld tokens of a lane stay in registers for the five looks at them: up to
// 8192 tokens of a block (cluster barriers empty L1).
constexpr int kHeld = 8;

template <int kCluster>
__global__ void __launch_bounds__(kSelThreads)
kv_evict_select_kernel(const SelectParams p) {
  __shared__ __align__(8) uint32_t hist[kSelBins];
  __shared__ __align__(8) uint32_t total[kCluster > 1 ? kSelBins : 2];
  __shared__ uint32_t warp_a[32], warp_b[32];
  __shared__ uint32_t sh_bin, sh_above, sh_more, sh_equal;
  chain_trigger();
  chain_wait();
  const int rank = blockIdx.x % kCluster, at_bh = blockIdx.x / kCluster;
  const int b = at_bh / p.Hkv, h = at_bh % p.Hkv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gtid = rank * kSelThreads + tid;
  constexpr int kAll = kCluster * kSelThreads;
  const int len = min(max(p.seq_lens[b], 0), p.width);
  const int kept = min(len, p.keep);
  const float* w = p.weights + b * p.w_ld_b + h * p.w_ld_h;
  int* out = p.kept + ((long long)b * p.Hkv + h) * p.keep;
  float* wo = p.w_out + ((long long)b * p.Hkv + h) * p.keep;
  if (h == 0 && gtid == 0) p.new_lens[b] = kept;
  for (int i = kept + gtid; i < p.keep; i += kAll) { out[i] = -1; wo[i] = 0.f; }
  if (len <= p.keep) {                                  // the whole cluster
    for (int i = gtid; i < len; i += kAll) { out[i] = i; wo[i] = w[i]; }
    return;
  }
  const int lo = p.sink, hi = len - p.recent;
  for (int i = gtid; i < p.sink; i += kAll) { out[i] = i; wo[i] = w[i]; }
  for (int i = gtid; i < p.recent; i += kAll) { out[p.keep - p.recent + i] = hi + i; wo[p.keep - p.recent + i] = w[hi + i]; }
  const int span = (hi - lo + kAll - 1) / kAll * 32;    // tokens of a warp
  const int s0 = min(lo + (rank * 32 + warp) * span, hi), s1 = min(s0 + span, hi);
  int room = p.keep - p.sink - p.recent;                // hi - lo = len - sink - recent > room >= 0
  uint32_t held[kHeld];
#pragma unroll
  for (int j = 0; j < kHeld; ++j) {
    const int i = s0 + 32 * j + lane;
    held[j] = i < s1 ? weight_key(w[i]) : 0u;
  }
  // look(first token of 32, this lane's token and key) over the span; lanes behind its end take part
  auto span_keys = [&](auto look) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
      if (s0 + 32 * j < s1) look(s0 + 32 * j + lane, held[j]);
#pragma unroll 2
    for (int i0 = s0 + 32 * kHeld; i0 < s1; i0 += 32) look(i0 + lane, i0 + lane < s1 ? weight_key(w[i0 + lane]) : 0u);
  };
  uint32_t prefix = 0, mask = 0;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < kSelBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    span_keys([&](int i, uint32_t key) {
      const bool hit = i < s1 && (key & mask) == prefix;
      const uint32_t bin = (key >> shift) & ((1u << bits) - 1u);
      // tokens that nothing looked at share one bin: a warp adds equal neighbours at once
      const uint32_t first = __shfl_sync(0xffffffffu, bin, 0);
      const uint32_t same = __ballot_sync(0xffffffffu, hit && bin == first);
      if (hit && bin != first) atomicAdd(&hist[bin], 1u);
      if (lane == 0 && same) atomicAdd(&hist[first], (uint32_t)__popc(same));
    });
    uint32_t c0, c1;                                     // two bins a thread
    if constexpr (kCluster > 1) {
      const int two = 2 * (rank * (kSelThreads / kCluster) + tid / kCluster), of = tid % kCluster;
      cluster_sync_all();
      uint2 c = ld_cluster_u32x2(&hist[two], of);
#pragma unroll
      for (int o = 1; o < kCluster; o <<= 1) {
        c.x += __shfl_xor_sync(0xffffffffu, c.x, o);
        c.y += __shfl_xor_sync(0xffffffffu, c.y, o);
      }
      st_cluster_u32x2(&total[two], of, c);
      cluster_sync_all();                                // and every block has read the others' counts
      c0 = total[2 * tid]; c1 = total[2 * tid + 1];
    } else {
      __syncthreads();
      c0 = hist[2 * tid]; c1 = hist[2 * tid + 1];
    }
    // the bin that holds the room-th largest: suffix sums over the bins
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
    const uint32_t behind = (uint32_t)__reduce_add_sync(0xffffffffu, lane > warp ? warp_a[lane] : 0u);
    above += behind;
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
  uint32_t more = 0, equal = 0;
  span_keys([&](int i, uint32_t key) {
    more += i < s1 && key > prefix;
    equal += i < s1 && key == prefix;
  });
  more = (uint32_t)__reduce_add_sync(0xffffffffu, more);
  equal = (uint32_t)__reduce_add_sync(0xffffffffu, equal);
  if (lane == 0) { warp_a[warp] = more; warp_b[warp] = equal; }
  __syncthreads();
  int at = p.sink + (int)__reduce_add_sync(0xffffffffu, lane < warp ? warp_a[lane] : 0u);
  int ties = (int)__reduce_add_sync(0xffffffffu, lane < warp ? warp_b[lane] : 0u);
  if constexpr (kCluster > 1) {
    if (warp == 31 && lane == 0) { sh_more = (uint32_t)(at - p.sink) + more; sh_equal = (uint32_t)ties + equal; }
    cluster_sync_all();
    for (int r = 0; r < rank; ++r) {
      at += (int)ld_cluster_u32(&sh_more, r);
      ties += (int)ld_cluster_u32(&sh_equal, r);
    }
  }
  at += min(ties, room);
  span_keys([&](int i, uint32_t key) {
    const bool eq = i < s1 && key == prefix;
    const uint32_t eqs = __ballot_sync(0xffffffffu, eq);
    const bool take = (i < s1 && key > prefix) || (eq && ties + __popc(eqs & ((1u << lane) - 1u)) < room);
    const uint32_t takes = __ballot_sync(0xffffffffu, take);
    const int to = at + __popc(takes & ((1u << lane) - 1u));
    if (take && to < p.keep - p.recent) { out[to] = i; wo[to] = w[i]; }
    at += __popc(takes);
    ties += __popc(eqs);
  });
  if constexpr (kCluster > 1) cluster_sync_all();        // no block leaves while another reads its shared memory
}

struct MoveParams {
  ScaledCache from;
  uint8_t* k; uint8_t* v; float* ks; float* vs;
  const int* tables; int bt_ld;
  const int* to; int to_ld;
  const int* kept; const int* new_lens;
  int keep, pages; long long units;
};

// A warp fills one page of one head's keys or values.  A kept value token's 16-byte columns hold its neighbours too: every source page is read
// once, as a whole, for all tokens that come from it, kAhead pages at a time.  (A warp for two pages, keys and values one after the other: 31
// instead of 20 us for one sequence's 4096 tokens.)  Eight blocks an SM: 1024 of them, that sequence's, run at once (six: 47 us for the call, not 45),
// for which heads of 128 spill 284 bytes a thread.
template <int D>
__global__ void __launch_bounds__(128, D == 256 ? 3 : 8)
kv_evict_move_kernel(const MoveParams p) {
  constexpr int V = D / 32;
  constexpr int kAhead = 2;      // four pages ahead take the registers of a third of the warps: 138 us a call, not 115 (32 x 4096 tokens to 1024)
  chain_trigger();
  chain_wait();
  const int lane = threadIdx.x & 31;
  unsigned u = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (u >= (unsigned)p.units) return;
  const ScaledCache& c = p.from;
  const bool is_k = (u & 1) == 0;
  u >>= 1;
  const int pg = (int)(u % (unsigned)p.pages);
  u /= (unsigned)p.pages;
  const int h = (int)(u % (unsigned)c.Hkv), b = (int)(u / (unsigned)c.Hkv);
  // lane r < 16: where token r of the new page comes from (loads side by side; positions behind the last token are -1)
  const long long at = ((long long)b * c.Hkv + h) * p.keep + pg * kScPage + lane;
  const int pos = lane < kScPage && pg * kScPage + lane < p.keep ? p.kept[at] : -1;
  const int to = p.to[(long long)b * p.to_ld + pg];
  const int live = min(p.new_lens[b] - pg * kScPage, kScPage);
  if (live <= 0 || to < 0 || to >= c.num_pages) return;
  int page = -1, off = 0;
  float scale = 0.f;
  if (lane < live && pos >= 0) {
    page = p.tables[(long long)b * p.bt_ld + pos / kScPage];
    off = pos % kScPage;
    if (page < 0 || page >= c.num_pages) page = -1;
    else scale = is_k ? c.ks[page * c.ks_ld + h * c.ks_h] : c.vs[page * c.vs_ld + h * c.vs_h];
  }
  const long long head = (long long)h * (kScPage * D), step = (long long)c.Hkv * (kScPage * D);
  const long long base = (long long)to * step + head;
  if (is_k) {
    Codes<V> codes[kScPage];
#pragma unroll
    for (int r = 0; r < kScPage; ++r) {
      const int pr = __shfl_sync(0xffffffffu, page, r), o = __shfl_sync(0xffffffffu, off, r);
#pragma unroll
      for (int i = 0; i < (V + 3) / 4; ++i) codes[r].w[i] = 0;
      if (pr >= 0) codes[r] = load_codes<V>(c.k + head + pr * step + o * D + lane * V);
    }
    float amax = 0.f;
#pragma unroll
    for (int r = 0; r < kScPage; ++r) {
      float x[V], m = 0.f;
      widen<V>(codes[r], x);
#pragma unroll
      for (int i = 0; i < V; ++i) m = fmaxf(m, fabsf(x[i]));
      amax = fmaxf(amax, m * __shfl_sync(0xffffffffu, scale, r));
    }
    const int e = block_exponent(warp_max(amax));
    const float by = scale * exact_pow2(-e);                     // a power of two: exact
#pragma unroll
    for (int r = 0; r < kScPage; ++r) {
      const float f = __shfl_sync(0xffffffffu, by, r);
      if (f != 1.f) {                                       // the same for all lanes
        float x[V];
        widen<V>(codes[r], x);
        codes[r] = narrow<V>(x, f);
      }
      store_codes<V>(p.k + base + r * D + lane * V, codes[r]);
    }
    if (lane == 0) p.ks[to * c.ks_ld + h * c.ks_h] = exact_pow2(e);
    return;
  }
  // values: the distinct source pages in order, first token of each marked
  const int before = __shfl_up_sync(0xffffffffu, page, 1);
  uint32_t leads = __ballot_sync(0xffffffffu, lane < kScPage && (lane == 0 || page != before));
  uint32_t word[V][4];                                      // sixteen tokens of each of the lane's channels
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) word[i][j] = 0;
#pragma unroll 1
  while (leads) {
    uint4 col[kAhead][V];
    uint32_t mine[kAhead];                                  // tokens of the new page that come from the source page
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      mine[a] = 0;
      if (leads) {
        const int r = __ffs(leads) - 1;
        leads &= leads - 1;
        const int end = leads ? __ffs(leads) - 1 : kScPage;
        const int pr = __shfl_sync(0xffffffffu, page, r);
        if (pr >= 0) {
          mine[a] = ((1u << end) - 1u) & ~((1u << r) - 1u);
#pragma unroll
          for (int i = 0; i < V; ++i) col[a][i] = reinterpret_cast<const uint4*>(c.v + head + pr * step)[i * 32 + lane];
        }
      }
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
#pragma unroll
      for (int r = 0; r < kScPage; ++r) {
        if (!((mine[a] >> r) & 1u)) continue;               // the same for all lanes
        const int o = __shfl_sync(0xffffffffu, off, r);
        // byte r & 3 of the word becomes byte o & 3 of the column's word o / 4
        const uint32_t pick = (0x3210u & ~(0xFu << (4 * (r & 3)))) | ((4u + (o & 3)) << (4 * (r & 3)));
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const uint32_t lo = (o & 4) ? col[a][i].y : col[a][i].x, hi = (o & 4) ? col[a][i].w : col[a][i].z;
          word[i][r >> 2] = __byte_perm(word[i][r >> 2], (o & 8) ? hi : lo, pick);
        }
      }
  }
  float amax = 0.f;
#pragma unroll
  for (int r = 0; r < kScPage; r += 2) {
    float m0 = 0.f, m1 = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 t = codes2_to_f32((word[i][r >> 2] >> (8 * (r & 3))) & 0xFFFFu);
      m0 = fmaxf(m0, fabsf(t.x));
      m1 = fmaxf(m1, fabsf(t.y));
    }
    amax = fmaxf(amax, fmaxf(m0 * __shfl_sync(0xffffffffu, scale, r), m1 * __shfl_sync(0xffffffffu, scale, r + 1)));
  }
  const int e = block_exponent(warp_max(amax));
  const float by = scale * exact_pow2(-e);
#pragma unroll
  for (int r = 0; r < kScPage; r += 2) {
    const float f0 = __shfl_sync(0xffffffffu, by, r), f1 = __shfl_sync(0xffffffffu, by, r + 1);
    if (f0 == 1.f && f1 == 1.f) continue;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 t = codes2_to_f32((word[i][r >> 2] >> (8 * (r & 3))) & 0xFFFFu);
      const uint32_t two = f32_to_codes2(t.x * f0, t.y * f1);
      word[i][r >> 2] = (r & 2) ? __byte_perm(word[i][r >> 2], two, 0x5410) : __byte_perm(word[i][r >> 2], two, 0x3254);
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    reinterpret_cast<uint4*>(p.v + base)[i * 32 + lane] = make_uint4(word[i][0], word[i][1], word[i][2], word[i][3]);
  if (lane == 0) p.vs[to * c.vs_ld + h * c.vs_h] = exact_pow2(e);
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
    if (p.rows_per_block == 1) return launched(launch_chain(kv_scaled_write_kernel<D, 1>, dim3(blocks), dim3(256), 0, st, p));
    return launched(launch_chain_if(false, kv_scaled_write_kernel<D, 4>, dim3(blocks), dim3(256), 0, st, p));
  }
};
template <int D>
struct Read {
  static int launch(const ScaledCache& c, const int* tables, int bt_ld, int bt_cols, const int* lens, int max_len, int pages, unsigned units,
                    __nv_bfloat16* k, __nv_bfloat16* v, cudaStream_t st) {
    return launched(launch_chain(kv_scaled_read_kernel<D>, dim3((unsigned)((units + 7) / 8)), dim3(256), 0, st, c, tables, bt_ld, bt_cols, lens, max_len,
                                 pages, units, k, v));
  }
};
template <int D>
struct Move {
  static int launch(const MoveParams& p, cudaStream_t st) {
    return launched(launch_chain(kv_evict_move_kernel<D>, dim3((unsigned)((p.units + 3) / 4)), dim3(128), 0, st, p));
  }
};

}  // namespace

// The entry points take their arguments as one record (all fields 8 bytes wide): a call from Python costs 0.6 us so, and 3 us as thirty
// converted arguments.  -1: sizes or alignment that the kernels do not take (16-token pages, heads of 64, 128 or 256, queries and norm
// weights on 16 bytes, keys and values on 2 * D / 32, rotary widths in sixteens); -20: a launch failed.
struct ScalesRecord { float* ks; long long ks_ld, ks_h; float* vs; long long vs_ld, vs_h; };

struct WriteRecord {
  const void* q; long long ldq; void* q_out; long long ldqo; const void* k; long long ldk; const void* v; long long ldv;
  const int* positions; const float* rope; const void* q_norm; const void* k_norm;
  void* k_cache; void* v_cache; ScalesRecord s;
  const int* slots; long long T, Hq, Hkv, D, rotary, num_pages, plus_one, norm_dim; double eps; void* stream;
};
extern "C" int atlas_kv_scaled_write(const void* record) {
  const WriteRecord& r = *static_cast<const WriteRecord*>(record);
  const int D = (int)r.D;
  if (r.T <= 0) return 0;
  if (D != 64 && D != 128 && D != 256) return -1;
  const int V = D / 32;
  if (r.T > 0x7fffffff || r.rotary < 0 || r.rotary > D || r.rotary % 16 || r.num_pages <= 0 || r.num_pages >= (1 << 27) || r.Hkv <= 0 || r.Hq < 0)
    return -1;
  if (r.ldk % V || r.ldv % V || !aligned(r.k, 2 * V) || !aligned(r.v, 2 * V) || !aligned(r.k_cache, 16) ||
      !aligned(r.v_cache, 16) || !aligned(r.rope, 16))
    return -1;
  if (r.Hq > 0 && (!aligned(r.q, 16) || !aligned(r.q_out, 16) || r.ldq % 8 || r.ldqo % 8)) return -1;
  if (!aligned(r.q_norm, 16) || !aligned(r.k_norm, 2 * V)) return -1;
  ScaledWriteParams p;
  p.q = (const __nv_bfloat16*)r.q; p.ldq = r.ldq; p.q_out = (__nv_bfloat16*)r.q_out; p.ldqo = r.ldqo;
  p.k = (const __nv_bfloat16*)r.k; p.ldk = r.ldk; p.v = (const __nv_bfloat16*)r.v; p.ldv = r.ldv;
  p.positions = r.positions; p.rope = r.rope; p.q_norm = (const __nv_bfloat16*)r.q_norm; p.k_norm = (const __nv_bfloat16*)r.k_norm;
  p.k_cache = (uint8_t*)r.k_cache; p.v_cache = (uint8_t*)r.v_cache;
  p.k_scale = r.s.ks; p.v_scale = r.s.vs; p.ks_ld = r.s.ks_ld; p.vs_ld = r.s.vs_ld; p.ks_h = (int)r.s.ks_h; p.vs_h = (int)r.s.vs_h;
  p.slots = r.slots; p.T = (int)r.T; p.Hq = (int)r.Hq; p.Hkv = (int)r.Hkv; p.rotary = (int)r.rotary; p.num_pages = (int)r.num_pages;
  p.plus_one = (int)r.plus_one; p.norm_dim = r.norm_dim > 0 ? (int)r.norm_dim : D; p.eps = (float)r.eps;
  // Up to 512 rows: one row a block, a warp per page, the plan of single tokens.  More are prompts: a page gets four warps, and one row in 16
  // begins a page; blocks of four or sixteen rows leave fewer blocks empty, but a mixed step's decode rows go through their block one after the
  // other, which a long prompt beside them hides.  The number of rows does not tell prompts from single tokens, and a prompt of 17 to 512 rows
  // pays for that (us, a warp per page and four):
  //   heads of 128   prompts of 32, 128, 512 rows 22.6 / 5.1, 22.9 / 5.3, 25.9 / 8.2   32, 128, 512 single tokens 4.6 / 11.3, 4.9 / 11.6, 8.5 / 19.5
  //   heads of 256   prompts of 32, 128, 512 rows 18.7 / 6.3, 18.9 / 6.3, 20.6 / 8.1   32, 128, 512 single tokens 4.6 / 17.0, 4.8 / 17.3, 9.9 / 26.4
  p.rows_per_block = p.T <= 512 ? 1 : p.T < 2048 ? 4 : 16;
  p.kv_blocks_x = (p.T + p.rows_per_block - 1) / p.rows_per_block;
  p.kv_blocks_y = p.rows_per_block == 1 ? (p.Hkv + 7) / 8 : (p.Hkv + 1) / 2;
  const int heads = 4 * 256 / D;                   // queries of a warp
  const long long q_units = r.T * ((p.Hq + heads - 1) / heads);
  const long long blocks = (long long)p.kv_blocks_x * p.kv_blocks_y + (q_units + 7) / 8;
  if (blocks > 0x7fffffffll / 8) return -1;
  return by_width<Write>(D, p, (unsigned)blocks, (cudaStream_t)r.stream);
}

struct ReadRecord {
  const void* k_cache; const void* v_cache; ScalesRecord s;
  const int* tables; long long bt_ld, bt_cols; const int* lens; long long B, max_len, Hkv, D, num_pages; void* k_out; void* v_out; void* stream;
};
extern "C" int atlas_kv_scaled_read(const void* record) {
  const ReadRecord& r = *static_cast<const ReadRecord*>(record);
  if (r.B <= 0 || r.max_len <= 0) return 0;
  if (!aligned(r.k_cache, 16) || !aligned(r.v_cache, 16) || !aligned(r.k_out, 16) || !aligned(r.v_out, 16) || r.bt_cols > (1 << 26) ||
      r.max_len > (1 << 30))
    return -1;
  const ScaledCache c{(const uint8_t*)r.k_cache, (const uint8_t*)r.v_cache, r.s.ks, r.s.vs, r.s.ks_ld, r.s.vs_ld, (int)r.s.ks_h, (int)r.s.vs_h,
                      (int)r.Hkv, (int)r.num_pages};
  const int pages = (int)((r.max_len + kScPage - 1) / kScPage);
  const long long units = 2ll * r.B * pages * r.Hkv;
  if (units > 0x7fffffffll) return -1;
  return by_width<Read>((int)r.D, c, r.tables, (int)r.bt_ld, (int)r.bt_cols, r.lens, (int)r.max_len, pages, (unsigned)units, (__nv_bfloat16*)r.k_out,
                        (__nv_bfloat16*)r.v_out, (cudaStream_t)r.stream);
}

struct EvictRecord {
  void* k_cache; void* v_cache; ScalesRecord s;
  const int* tables; long long bt_ld; const int* seq_lens; const float* weights; long long w_ld_b, w_ld_h, width;
  long long B, Hkv, D, num_pages, keep, sink, recent; const int* to; long long to_ld; int* new_lens; int* kept; float* w_out; long long sms; void* stream;
};
extern "C" int atlas_kv_evict(const void* record) {
  const EvictRecord& r = *static_cast<const EvictRecord*>(record);
  if (r.B <= 0) return 0;
  if (r.keep <= 0 || r.sink < 0 || r.recent < 0 || r.sink + r.recent > r.keep || r.keep > (1 << 30) || !aligned(r.k_cache, 16) ||
      !aligned(r.v_cache, 16) || r.B * r.Hkv > 0x7fffffffll)
    return -1;
  if (r.D != 64 && r.D != 128 && r.D != 256) return -1;
  cudaStream_t st = (cudaStream_t)r.stream;
  const int Hkv = (int)r.Hkv, keep = (int)r.keep;
  SelectParams s{r.weights, r.w_ld_b, r.w_ld_h, r.seq_lens, r.new_lens, r.kept, r.w_out, Hkv, keep, (int)r.sink, (int)r.recent, (int)r.width};
  MoveParams m;
  m.from = ScaledCache{(const uint8_t*)r.k_cache, (const uint8_t*)r.v_cache, r.s.ks, r.s.vs, r.s.ks_ld, r.s.vs_ld, (int)r.s.ks_h, (int)r.s.vs_h, Hkv,
                       (int)r.num_pages};
  m.k = (uint8_t*)r.k_cache; m.v = (uint8_t*)r.v_cache; m.ks = r.s.ks; m.vs = r.s.vs;
  m.tables = r.tables; m.bt_ld = (int)r.bt_ld; m.to = r.to; m.to_ld = (int)r.to_ld; m.kept = r.kept; m.new_lens = r.new_lens; m.keep = keep;
  const long long longest = r.width < r.keep ? r.width : r.keep;
  m.pages = (int)((longest + kScPage - 1) / kScPage);
  m.units = 2ll * r.B * Hkv * m.pages;
  if (m.units > 0x7fffffffll || r.B * Hkv > 0x7fffffffll / 8) return -1;
  // As many blocks a head, up to eight, as there are SMs for and 2048 tokens each: a block has an SM to itself, and a second wave of
  // clusters doubles the time (256 heads of 4096 tokens: 19 us on a block each, 470 on clusters of eight).
  int n = 1;
  while (n < 8 && r.B * Hkv * n * 2 <= r.sms && r.width >= 4096ll * n) n *= 2;
  const dim3 blocks((unsigned)(r.B * Hkv * n)), threads(kSelThreads);
  const cudaError_t e = n == 8   ? launch_chain_cluster(true, 8, kv_evict_select_kernel<8>, blocks, threads, 0, st, s)
                        : n == 4 ? launch_chain_cluster(true, 4, kv_evict_select_kernel<4>, blocks, threads, 0, st, s)
                        : n == 2 ? launch_chain_cluster(true, 2, kv_evict_select_kernel<2>, blocks, threads, 0, st, s)
                                 : launch_chain(kv_evict_select_kernel<1>, blocks, threads, 0, st, s);
  const int rc = launched(e);
  if (rc || m.units == 0) return rc;
  return by_width<Move>((int)r.D, m, st);
}

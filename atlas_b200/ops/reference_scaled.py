"""Plain forms of the FP8 cache with a power-of-two scale per (block, head), in fp32 (``csrc/kv_scaled.cu`` has the formulas)."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
LOW, HIGH = -60, 60


def block_scale(amax: torch.Tensor) -> torch.Tensor:
    """The smallest ``2^e``, ``-60 <= e <= 60``, with ``amax <= 448 * 2^e``."""
    m, x = torch.frexp(amax.float())                              # 448 = 7/8 * 2^9
    e = torch.where(m <= 0.875, x - 9, x - 8)
    e = torch.where(amax > 0, e, torch.full_like(e, LOW))
    e = torch.where(torch.isinf(amax), torch.full_like(e, HIGH), e)
    return torch.ldexp(torch.ones_like(amax, dtype=torch.float32), e.clamp(LOW, HIGH))


def codes(x: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    return (x.float() / scale).clamp(-FP8_MAX, FP8_MAX).to(FP8)


def _turn(x: torch.Tensor, positions, rope_cache, rotary_dim: int, w, eps: float, plus_one: bool, norm_dim: int) -> torch.Tensor:
    """Head norm and rotation in fp32, nothing rounded on the way."""
    x = x.float()
    if w is not None:
        w = w.float() + 1.0 if plus_one else w.float()
        x = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / (norm_dim or x.shape[-1]) + eps) * w
    if not rotary_dim:
        return x
    half = rotary_dim // 2
    cs = rope_cache[positions.long()][:, None]
    c, s, a, b = cs[..., :half], cs[..., half:], x[..., :half], x[..., half:rotary_dim]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., rotary_dim:]], -1)


def qk_norm_rope_kv_write(q, k, v, positions, rope_cache, rotary_dim, k_cache, v_cache, slot_mapping, k_scale, v_scale, q_norm_w=None,
                          k_norm_w=None, eps=1e-6, norm_plus_one=False, norm_dim=0) -> torch.Tensor:
    out = _turn(q, positions, rope_cache, rotary_dim, q_norm_w, eps, norm_plus_one, norm_dim).to(q.dtype)
    kf = _turn(k, positions, rope_cache, rotary_dim, k_norm_w, eps, norm_plus_one, norm_dim)
    bs = k_cache.shape[1]
    slots = slot_mapping.tolist()
    t = 0
    while t < len(slots):
        s = slots[t]
        if s < 0 or s >= k_cache.shape[0] * bs:                                   # padding, or outside of the pool
            t += 1
            continue
        blk, off, n = s // bs, s % bs, 1
        while t + n < len(slots) and off + n < bs and slots[t + n] == s + n:
            n += 1
        for x, cache, scales in ((kf, k_cache, k_scale), (v.float(), v_cache, v_scale)):
            rows = x[t:t + n]                                                     # [n, Hkv, D]
            new = block_scale(torch.nan_to_num(rows.abs(), nan=0.0, posinf=float("inf")).amax((0, 2)))
            if off:
                old = scales[blk].clone()
                new = torch.maximum(new, old)
                shift = (old / new)[None, :, None]
                cache[blk, :off] = (cache[blk, :off].float() * shift).to(FP8)
            cache[blk, off:off + n] = codes(rows, new[None, :, None])
            scales[blk] = new
        t += n
    return out


def values(cache: torch.Tensor, scales: torch.Tensor, blocks: torch.Tensor) -> torch.Tensor:
    """fp32 ``[n * block, Hkv, D]`` of the given blocks; zeros where one lies outside of the pool."""
    there = pooled(blocks, cache.shape[0])
    at = torch.where(there, blocks, torch.zeros_like(blocks))
    raw = cache.view(torch.uint8)[at].view(FP8).float()
    x = torch.where(there[:, None, None, None], raw * scales[at][:, None, :, None], torch.zeros((), device=raw.device))
    return x.reshape(-1, *raw.shape[2:])


def pooled(blocks: torch.Tensor, num_blocks: int) -> torch.Tensor:
    return (blocks >= 0) & (blocks < num_blocks)


def kv_read(k_cache, v_cache, block_tables, seq_lens, max_len: int, k_scale, v_scale) -> Tuple[torch.Tensor, torch.Tensor]:
    nb, bs, hkv, d = k_cache.shape
    B = block_tables.shape[0]
    out = [torch.zeros(B, max_len, hkv, d, dtype=torch.bfloat16, device=k_cache.device) for _ in range(2)]
    for b, n in enumerate(seq_lens.tolist()):
        n = min(n, max_len)
        blocks = block_tables[b, :(n + bs - 1) // bs].long()
        for o, cache, scales in zip(out, (k_cache, v_cache), (k_scale, v_scale)):
            o[b, :n] = values(cache, scales, blocks)[:n].to(torch.bfloat16)
    return out[0], out[1]


def paged_attention(q, k_cache, v_cache, block_tables, seq_lens, query_start_loc, scale, k_scale, v_scale, sliding_window: Optional[int] = None,
                    weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    T, Hq, D = q.shape
    nb, bs, hkv, _ = k_cache.shape
    out = torch.zeros_like(q)
    starts = query_start_loc.tolist()
    for b, L in enumerate(seq_lens.tolist()):
        r0, r1 = starts[b], starts[b + 1]
        n = r1 - r0
        if n <= 0 or L <= 0:
            continue
        blocks = block_tables[b, :(L + bs - 1) // bs].long()
        kk, vv = values(k_cache, k_scale, blocks)[:L], values(v_cache, v_scale, blocks)[:L]
        s = torch.einsum("qhgd,khd->hgqk", q[r0:r1].float().view(n, hkv, Hq // hkv, D), kk) * scale
        qpos, kpos = torch.arange(L - n, L, device=q.device)[:, None], torch.arange(L, device=q.device)[None]
        mask = (kpos <= qpos) & pooled(blocks, nb).repeat_interleave(bs)[None, :L]       # a block outside of the pool is skipped
        if sliding_window:
            mask &= kpos > qpos - sliding_window
        p = torch.softmax(s.masked_fill(~mask, float("-inf")), -1)
        p = torch.where(mask.any(-1)[:, None], p, torch.zeros((), device=q.device))      # a row that sees nothing: zeros
        out[r0:r1] = torch.einsum("hgqk,khd->qhgd", p, vv).reshape(n, Hq, D).to(q.dtype)
        if weights is not None:
            weights[b, :, :L] += p.sum((1, 2))
    return out


def kv_evict(k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens, weights, keep: int, new_tables, sink: int, recent: int):
    nb, bs, hkv, d = k_cache.shape
    B = block_tables.shape[0]
    dev = k_cache.device
    kept = torch.full((B, hkv, keep), -1, dtype=torch.int32, device=dev)
    out_w = torch.zeros(B, hkv, keep, dtype=torch.float32, device=dev)
    lens = seq_lens.clamp(max=keep).to(torch.int32)
    for b, L in enumerate(seq_lens.tolist()):
        n = min(L, keep)
        if n <= 0:
            continue
        w = weights[b, :, :L]
        if L <= keep:
            pos = torch.arange(L, device=dev).expand(hkv, L)
        else:
            room = keep - sink - recent
            mid = w[:, sink:L - recent]
            order = torch.sort(torch.where(mid.isnan(), torch.full_like(mid, float("-inf")), mid), dim=1, descending=True, stable=True).indices
            last = torch.sort(mid.isnan().gather(1, order).to(torch.uint8), dim=1, stable=True).indices             # NaN below -inf, too
            best = order.gather(1, last)[:, :room] + sink
            ends = torch.cat([torch.arange(sink, device=dev), torch.arange(L - recent, L, device=dev)]).expand(hkv, -1)
            pos = torch.sort(torch.cat([best, ends], 1), dim=1).values
        kept[b, :, :n] = pos.to(torch.int32)
        out_w[b, :, :n] = weights[b, :, :L].gather(1, pos)
        blocks = block_tables[b, :(L + bs - 1) // bs].long()
        for cache, scales in ((k_cache, k_scale), (v_cache, v_scale)):
            x = values(cache, scales, blocks)[:L].transpose(0, 1).gather(1, pos[:, :, None].expand(-1, -1, d))      # [Hkv, n, D]
            for i in range((n + bs - 1) // bs):
                part = x[:, i * bs:(i + 1) * bs]
                s = block_scale(part.abs().amax((1, 2)))
                to = int(new_tables[b, i])
                page = torch.zeros(bs, hkv, d, dtype=FP8, device=dev)
                page[:part.shape[1]] = codes(part, s[:, None, None]).transpose(0, 1)
                cache[to] = page
                scales[to] = s
    return lens, kept, out_w

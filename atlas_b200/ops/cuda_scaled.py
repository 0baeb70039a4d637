"""Bindings of the FP8 cache with a power-of-two scale per (16-token block, head): ``csrc/kv_scaled.cu``, ``csrc/attention_scaled.cu``,
``csrc/attention_scaled_tc.cu``.  Every call launches on the current stream of its tensors' device; workspaces come from the caching
allocator, so calls on several streams and captured graphs do not share any."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import checked, cuda as K

_vp, _ll, _i, _f = C.c_void_p, C.c_longlong, C.c_int, C.c_float
BLOCK = 16
HEAD_DIMS = (64, 128, 256)


def _lib():
    L = K.lib()
    if not getattr(L, "_scaled_bound", False):
        L.atlas_kv_scaled_write.argtypes = [_vp, _ll, _vp, _ll, _vp, _ll, _vp, _ll, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _ll, _i, _vp, _ll, _i, _vp,
                                            _i, _i, _i, _i, _i, _i, _i, _i, _f, _vp]
        L.atlas_kv_scaled_read.argtypes = [_vp, _vp, _vp, _ll, _i, _vp, _ll, _i, _vp, _i, _i, _vp, _i, _i, _i, _i, _i, _vp, _vp, _vp]
        L.atlas_kv_evict.argtypes = [_vp, _vp, _vp, _ll, _i, _vp, _ll, _i, _vp, _i, _vp, _vp, _ll, _ll, _i, _i, _i, _i, _i, _i, _i, _i, _vp, _i,
                                     _vp, _vp, _vp, _vp]
        L.atlas_attn_scaled_decode_plan.argtypes = [_i, _i, _i, _i, _i, C.POINTER(_i), C.POINTER(_i), C.POINTER(_ll)]
        L.atlas_attn_scaled_decode.argtypes = [_vp, _ll, _vp, _ll, _vp, _vp, _vp, _ll, _i, _vp, _ll, _i, _vp, _i, _i, _vp, _vp, _i, _f, _i, _i, _i, _i,
                                               _i, _i, _i, _vp, _vp, _vp, _ll, _vp, _vp, _ll, _ll, _vp, _vp]
        L.atlas_attn_scaled_chunk.argtypes = [_vp, _ll, _vp, _ll, _vp, _vp, _vp, _ll, _i, _vp, _ll, _i, _vp, _i, _i, _vp, _vp, _vp, _vp, _i, _i, _f, _i,
                                              _i, _i, _i, _i, _vp, _vp, _vp]
        L.atlas_attn_scaled_chunk_weigh.argtypes = [_vp, _ll, _vp, _vp, _ll, _i, _vp, _i, _i, _vp, _vp, _vp, _vp, _i, _i, _f, _i, _i, _i, _i, _i, _vp,
                                                    _vp, _ll, _ll, _i, _vp, _vp]
        L._scaled_bound = True
    return L


def check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale, v_scale) -> Tuple[int, int, int]:
    """(blocks, heads, head width) of a block-scaled cache, or the error of what does not fit."""
    if not (isinstance(k_scale, torch.Tensor) and isinstance(v_scale, torch.Tensor)):
        raise K.KernelError("a block-scaled cache takes a scale tensor for the keys and one for the values")
    K._kv_layout_ok(k_cache, v_cache)
    nb, bs, hkv, d = k_cache.shape
    if k_cache.dtype != K.FP8 or v_cache.dtype != K.FP8 or v_cache.shape != k_cache.shape:
        raise K.KernelError("block scales belong to an FP8 (e4m3) cache of keys and values of one size")
    if bs != BLOCK or d not in HEAD_DIMS:
        raise K.KernelError(f"block scales take blocks of {BLOCK} tokens and heads of 64, 128 or 256, not {bs} and {d}")
    for s in (k_scale, v_scale):
        if s.dtype != torch.float32 or tuple(s.shape) != (nb, hkv) or s.device != k_cache.device or s.stride(1) >= 1 << 31:
            raise K.KernelError(f"block scales are fp32 [{nb}, {hkv}] beside the cache")
    if v_cache.device != k_cache.device:
        raise K.KernelError("keys and values of a cache are on one device")
    return nb, hkv, d


def _int_rows(t: torch.Tensor, what: str, device, dims: int) -> torch.Tensor:
    if t.dtype != torch.int32 or t.dim() != dims or t.device != device or (t.numel() and t.stride(-1) != 1):
        raise K.KernelError(f"{what}: int32 with {dims} dimension{'s' if dims > 1 else ''} on the cache's device, rows contiguous")
    return t


def _heads(x: torch.Tensor, what: str, device, d: int) -> None:
    if x.dtype != torch.bfloat16 or x.dim() != 3 or x.shape[2] != d or x.device != device:
        raise K.KernelError(f"{what}: bf16 [rows, heads, {d}] on the cache's device")
    if x.numel() and (x.stride(2) != 1 or x.stride(1) != d):
        raise K.KernelError(f"{what}: the heads of a row are contiguous")


def _scales(k_scale, v_scale):
    return (k_scale.data_ptr(), k_scale.stride(0), k_scale.stride(1), v_scale.data_ptr(), v_scale.stride(0), v_scale.stride(1))


def _run(rc: int, what: str) -> None:
    if rc == -1:
        raise K.KernelError(f"{what}: sizes or alignment that the kernel does not take")
    K._check(rc, what)


def alloc_kv_scales(num_blocks: int, hkv: int, device) -> Tuple[torch.Tensor, torch.Tensor]:
    """Scales of a cache, ones: keys and values of a (block, head) side by side, since attention reads them together."""
    both = torch.ones(num_blocks, hkv, 2, dtype=torch.float32, device=device)
    return both[..., 0], both[..., 1]


def qk_norm_rope_kv_write(q, k, v, positions, rope_cache, rotary_dim, k_cache, v_cache, slot_mapping, k_scale, v_scale, q_norm_w=None,
                          k_norm_w=None, eps=1e-6, norm_plus_one=False, norm_dim=0) -> torch.Tensor:
    nb, hkv, d = check_cache(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    T, hq = q.shape[0], q.shape[1]
    for x, what in ((q, "queries"), (k, "keys"), (v, "values")):
        _heads(x, what, dev, d)
        if x.shape[0] != T:
            raise K.KernelError(f"{what}: {x.shape[0]} rows beside {T} queries")
    if k.shape[1] != hkv or v.shape[1] != hkv:
        raise K.KernelError(f"the cache has {hkv} heads, keys and values {k.shape[1]} and {v.shape[1]}")
    _int_rows(slot_mapping, "slots", dev, 1)
    if slot_mapping.shape[0] != T:
        raise K.KernelError(f"{slot_mapping.shape[0]} slots for {T} rows")
    if rotary_dim:
        _int_rows(positions, "positions", dev, 1)
        if rotary_dim < 0 or rotary_dim > d or rotary_dim % (d // 16):
            raise K.KernelError(f"the rotated width of {d}-wide heads is a multiple of {d // 16}, at most {d}, not {rotary_dim}")
        if positions.shape[0] != T or rope_cache.dtype != torch.float32 or rope_cache.dim() != 2 or rope_cache.shape[1] != rotary_dim \
                or not rope_cache.is_contiguous() or rope_cache.device != dev:
            raise K.KernelError("rotation: a position per row and an fp32 [positions, rotary_dim] table beside the cache")
    if (q_norm_w is None) != (k_norm_w is None):
        raise K.KernelError("head norms come for queries and keys together")
    for w in (q_norm_w, k_norm_w):
        if w is not None and (w.dtype != torch.bfloat16 or w.shape != (d,) or not w.is_contiguous() or w.device != dev):
            raise K.KernelError(f"head norm weights are bf16 [{d}]")
    out = torch.empty(T, hq, d, dtype=q.dtype, device=dev)
    if T == 0:
        return out
    if checked.ENABLED:
        checked.kv_write(slot_mapping, positions, nb, BLOCK, rope_cache.shape[0] if rotary_dim else 0)
        checked.block_runs(slot_mapping, BLOCK)
    with torch.cuda.device(dev):
        K._dev(q)
        _run(_lib().atlas_kv_scaled_write(q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(),
                                          v.stride(0), K._ptr(positions) if rotary_dim else None, rope_cache.data_ptr() if rotary_dim else None,
                                          K._ptr(q_norm_w), K._ptr(k_norm_w), k_cache.data_ptr(), v_cache.data_ptr(), *_scales(k_scale, v_scale),
                                          slot_mapping.data_ptr(), T, hq, hkv, d, rotary_dim, nb, 1 if norm_plus_one else 0, int(norm_dim or d),
                                          float(eps), K._stream()), "kv_scaled_write")
    return out


def kv_read(k_cache, v_cache, block_tables, seq_lens, max_len: int, k_scale, v_scale) -> Tuple[torch.Tensor, torch.Tensor]:
    nb, hkv, d = check_cache(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    _int_rows(block_tables, "block tables", dev, 2)
    _int_rows(seq_lens, "sequence lengths", dev, 1)
    B = block_tables.shape[0]
    if seq_lens.shape[0] != B or max_len < 0:
        raise K.KernelError(f"{seq_lens.shape[0]} lengths for {B} block tables, {max_len} tokens of each")
    out = torch.empty(2, B, max_len, hkv, d, dtype=torch.bfloat16, device=dev)
    if out.numel():
        with torch.cuda.device(dev):
            K._dev(k_cache)
            _run(_lib().atlas_kv_scaled_read(k_cache.data_ptr(), v_cache.data_ptr(), *_scales(k_scale, v_scale), block_tables.data_ptr(),
                                             block_tables.stride(0), block_tables.shape[1], seq_lens.data_ptr(), B, max_len, hkv, d, nb, out[0].data_ptr(),
                                             out[1].data_ptr(), K._stream()), "kv_scaled_read")
    return out[0], out[1]


def kv_evict(k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens, weights, keep: int, new_tables, sink: int, recent: int):
    nb, hkv, d = check_cache(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    for t, what, n in ((block_tables, "block tables", 2), (new_tables, "new block tables", 2), (seq_lens, "sequence lengths", 1)):
        _int_rows(t, what, dev, n)
    B = block_tables.shape[0]
    if keep < 1 or sink < 0 or recent < 0 or sink + recent > keep:
        raise K.KernelError(f"keeping {keep} tokens of which the first {sink} and the last {recent} are fixed")
    if weights.dtype != torch.float32 or weights.dim() != 3 or weights.shape[:2] != (B, hkv) or weights.device != dev \
            or (weights.numel() and weights.stride(2) != 1):
        raise K.KernelError(f"weights are fp32 [{B}, {hkv}, tokens] beside the cache, tokens contiguous")
    width = min(weights.shape[2], block_tables.shape[1] * BLOCK)      # no sequence is longer
    need = (min(keep, width) + BLOCK - 1) // BLOCK
    if seq_lens.shape[0] != B or new_tables.shape[0] != B or new_tables.shape[1] < need:
        raise K.KernelError(f"{B} sequences that keep up to {min(keep, width)} tokens need their lengths and new block tables of {need} columns")
    lens = torch.empty(B, dtype=torch.int32, device=dev)
    kept = torch.empty(B, hkv, keep, dtype=torch.int32, device=dev)
    out_w = torch.empty(B, hkv, keep, dtype=torch.float32, device=dev)
    if B == 0:
        return lens, kept, out_w
    if checked.ENABLED:
        checked.evict(block_tables, seq_lens, new_tables, nb, BLOCK, keep, width)
    with torch.cuda.device(dev):
        K._dev(k_cache)
        _run(_lib().atlas_kv_evict(k_cache.data_ptr(), v_cache.data_ptr(), *_scales(k_scale, v_scale), block_tables.data_ptr(),
                                   block_tables.stride(0), seq_lens.data_ptr(), weights.data_ptr(), weights.stride(0), weights.stride(1), width,
                                   B, hkv, d, nb, keep, sink, recent, new_tables.data_ptr(), new_tables.stride(0), lens.data_ptr(),
                                   kept.data_ptr(), out_w.data_ptr(), K._stream()), "kv_evict")
    return lens, kept, out_w


def _weigh_tiles(batch, nd: int, device):
    """Tiles of 128 cached tokens of the chunk sequences, those with the most rows first: (device [2, n], n)."""
    tiles = getattr(batch, "_weigh_tiles", None)
    if tiles is None:
        work = []
        for i in range(nd, batch.num_seqs):
            n, rows = batch.seq_lens_host[i], batch.query_lens_host[i]
            if rows:
                work += [(-(rows - max(0, k0 - (n - rows))), i, k0) for k0 in range(0, n, 128)]
        work.sort()
        host = torch.tensor([[w[1] for w in work], [w[2] for w in work]], dtype=torch.int32).pin_memory()
        tiles = batch._weigh_tiles = (host.to(device, non_blocking=True), len(work))
    return tiles


def paged_attention(q, k_cache, v_cache, batch, scale, k_scale, v_scale, sliding_window: Optional[int] = None,
                    weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    nb, hkv, d = check_cache(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    _heads(q, "queries", dev, d)
    T, hq = q.shape[0], q.shape[1]
    if hq % hkv or hq // hkv > 128:
        raise K.KernelError(f"{hq} query heads over {hkv} key heads: up to 128 for each")
    if q.stride(0) % 8 or q.data_ptr() % 16:
        raise K.KernelError("queries start on 16 bytes in every row")
    bt, lens, starts = batch.block_tables, batch.seq_lens, batch.query_start_loc
    _int_rows(bt, "block tables", dev, 2)
    _int_rows(lens, "sequence lengths", dev, 1)
    _int_rows(starts, "query starts", dev, 1)
    window, nd, B = int(sliding_window or 0), batch.num_decodes, batch.num_seqs
    if window < 0 or bt.shape[0] < B or starts.shape[0] < B + 1 or not 0 <= nd <= B or T < nd:
        raise K.KernelError("attention: a block table, a length and a start for every sequence, a row for every decode, no negative window")
    if weights is not None and (weights.dtype != torch.float32 or weights.dim() != 3 or tuple(weights.shape[:2]) != (B, hkv) or weights.device != dev
                                or weights.stride(2) != 1 or weights.shape[2] < batch.max_seq_len):
        raise K.KernelError(f"weights are fp32 [{B}, {hkv}, at least {batch.max_seq_len}] beside the cache, tokens contiguous")
    out = torch.empty(T, hq, d, dtype=q.dtype, device=dev)
    if T == 0 or B == 0:
        return out
    if checked.ENABLED:
        checked.paged_read(bt, lens, nb, BLOCK)
    L = _lib()
    with torch.cuda.device(dev):
        index = K._dev(q)
        st, status, sms = K._stream(), K._status_ptr[index], K._num_sms[index]
        new = lambda *shape: torch.empty(shape, dtype=torch.float32, device=dev)
        sums = (None, 0, 0) if weights is None else (weights.data_ptr(), weights.stride(0), weights.stride(1))
        if nd > 0:
            blocks, cols, pieces = _i(), _i(), _ll()
            _run(L.atlas_attn_scaled_decode_plan(nd, hq, hkv, batch.max_seq_len, sms, C.byref(blocks), C.byref(cols), C.byref(pieces)),
                 "attn_scaled_decode")
            part_o, part_ml = new(pieces.value * d * cols.value), new(pieces.value * cols.value * 2)
            scores = ml = None
            width = 0
            if weights is not None:
                width = weights.shape[2]
                scores, ml = new(nd * hkv, width, (hq // hkv + 1) // 2 * 2), new(nd, hq, 2)
            _run(L.atlas_attn_scaled_decode(q.data_ptr(), q.stride(0), out.data_ptr(), hq * d, k_cache.data_ptr(), v_cache.data_ptr(),
                                            *_scales(k_scale, v_scale), bt.data_ptr(), bt.stride(0), bt.shape[1], lens.data_ptr(), starts.data_ptr(), nd,
                                            float(scale), hq, hkv, d, window, nb, batch.max_seq_len, sms, part_o.data_ptr(), part_ml.data_ptr(),
                                            K._ptr(scores), width, K._ptr(ml), *sums, status, st), "attn_scaled_decode")
        if B > nd:
            tiles, n, _ = K._tc_tiles(q, batch, nd, 128 // (hq // hkv))
            ml = new(T, hq, 2) if weights is not None else None
            _run(L.atlas_attn_scaled_chunk(q.data_ptr(), q.stride(0), out.data_ptr(), hq * d, k_cache.data_ptr(), v_cache.data_ptr(),
                                           *_scales(k_scale, v_scale), bt.data_ptr(), bt.stride(0), bt.shape[1], lens.data_ptr(), starts.data_ptr(),
                                           tiles[0].data_ptr(), tiles[1].data_ptr(), n, T, float(scale), hq, hkv, d, window, nb, K._ptr(ml), status,
                                           st), "attn_scaled_chunk")
            if weights is not None:
                tiles, n = _weigh_tiles(batch, nd, dev)
                _run(L.atlas_attn_scaled_chunk_weigh(q.data_ptr(), q.stride(0), k_cache.data_ptr(), *_scales(k_scale, v_scale)[:3], bt.data_ptr(),
                                                     bt.stride(0), bt.shape[1], lens.data_ptr(), starts.data_ptr(), tiles[0].data_ptr(), tiles[1].data_ptr(), n,
                                                     T, float(scale), hq, hkv, d, window, nb, ml.data_ptr(), *sums, weights.shape[2], status, st),
                     "attn_scaled_chunk_weigh")
    return out

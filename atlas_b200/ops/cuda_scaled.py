"""Bindings of the FP8 cache with a power-of-two scale per (16-token block, head): ``csrc/kv_scaled.cu``, ``csrc/attention_scaled.cu``,
``csrc/attention_scaled_tc.cu``.

Every call launches on the current stream of its tensors' device.  Workspaces come from the caching allocator, so calls on several streams
and captured graphs share none.  A call's arguments go over as one packed record (a decode step of one sequence costs the host 15 us so, and
45 us with one converted argument each, the stream looked up through ``torch.cuda.current_stream`` and a device guard around every launch)."""
from __future__ import annotations

import contextlib
import ctypes as C
import struct
from typing import Optional, Tuple

import torch

from . import checked, cuda as K

BLOCK = 16
HEAD_DIMS = (64, 128, 256)
WARPS, LEAST = 16, 2               # of scaled_decode_kernel: most warps of a block, pages worth a warp
_F32, _BF16, _I32, _FP8 = torch.float32, torch.bfloat16, torch.int32, torch.float8_e4m3fn

# records of the entry points, in the order of their C structs: integers and pointers, one double
_WRITE = struct.Struct("=29qdq")
_READ = struct.Struct("=20q")
_EVICT = struct.Struct("=29q")
_DECODE = struct.Struct("=33qd2q")
_CHUNK = struct.Struct("=39qd2q")
_calls: dict = {}
_HERE = contextlib.nullcontext()


def _call(name: str, record: bytes, what: str) -> None:
    f = _calls.get(name)
    if f is None:
        f = getattr(K.lib(), name)
        f.argtypes = [C.c_char_p]
        _calls[name] = f
    rc = f(record)
    if rc == -1:
        raise K.KernelError(f"{what}: sizes or alignment that the kernel does not take")
    K._check(rc, what)


def _place(t: torch.Tensor):
    """(guard for launches beside ``t``, device index, its current stream)."""
    i = t.get_device()
    if i < 0:
        raise K.KernelError("the kernels take tensors on a GPU")
    if i not in K._status_ptr:
        K._dev(t)
    return _HERE if torch._C._cuda_getDevice() == i else torch.cuda.device(i), i, torch._C._cuda_getCurrentRawStream(i)


def check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale, v_scale) -> Tuple[int, int, int]:
    """(blocks, heads, head width) of a block-scaled cache, or the error of what does not fit."""
    if not (isinstance(k_scale, torch.Tensor) and isinstance(v_scale, torch.Tensor)):
        raise K.KernelError("a block-scaled cache takes a scale tensor for the keys and one for the values")
    shape, dev = k_cache.shape, k_cache.get_device()
    if len(shape) != 4:
        raise K.KernelError("a cache has four dimensions: blocks, tokens, heads, channels")
    nb, bs, hkv, d = shape
    if hkv < 1:
        raise K.KernelError("a cache has at least one head")
    if k_cache.dtype != _FP8 or v_cache.dtype != _FP8 or v_cache.shape != shape:
        raise K.KernelError("block scales belong to an FP8 (e4m3) cache of keys and values of one size")
    if bs != BLOCK or d not in HEAD_DIMS:
        raise K.KernelError(f"block scales take blocks of {BLOCK} tokens and heads of 64, 128 or 256, not {bs} and {d}")
    page = BLOCK * d
    if k_cache.stride() != (hkv * page, d, page, 1) or v_cache.stride() != (hkv * page, 1, page, BLOCK):
        raise K.KernelError("KV cache is not in the kernel layout (allocate it with ops.cuda.alloc_kv_cache)")
    if v_cache.get_device() != dev:
        raise K.KernelError("keys and values of a cache are on one device")
    for s in (k_scale, v_scale):
        if s.dtype != _F32 or s.shape != (nb, hkv) or s.get_device() != dev or s.stride(1) >= 1 << 31:
            raise K.KernelError(f"block scales are fp32 [{nb}, {hkv}] beside the cache")
    return nb, hkv, d


def _apart(t: torch.Tensor) -> bool:
    """Whether all elements have places of their own (a view that was not interleaved with itself)."""
    reach = 0
    for step, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if step <= reach:
            return False
        reach += step * (size - 1)
    return True


def _writable(k_cache, v_cache, k_scale, v_scale) -> None:
    """What a call writes is not written through two places at once."""
    st = k_scale.stride()
    own = st[1] == 2 and st[0] == 2 * k_scale.shape[1] and v_scale.stride() == st or (_apart(k_scale) and _apart(v_scale))      # first: alloc_kv_scales
    if not own or k_scale.data_ptr() == v_scale.data_ptr() or k_cache.data_ptr() == v_cache.data_ptr():
        raise K.KernelError("keys, values and their scales have places of their own (allocate the scales with ops.alloc_kv_scales)")


def _ints(t: torch.Tensor, what: str, dev: int, dims: int) -> None:
    if t.dtype != _I32 or t.dim() != dims or t.get_device() != dev or (t.stride(-1) != 1 and t.numel() > 1):
        raise K.KernelError(f"{what}: int32 with {dims} dimension{'s' if dims > 1 else ''} on the cache's device, rows contiguous")


def _heads(x: torch.Tensor, what: str, dev: int, d: int) -> None:
    if x.dtype != _BF16 or x.dim() != 3 or x.shape[2] != d or x.get_device() != dev:
        raise K.KernelError(f"{what}: bf16 [rows, heads, {d}] on the cache's device")
    st = x.stride()
    if (st[2] != 1 or st[1] != d) and x.numel():
        raise K.KernelError(f"{what}: the heads of a row are contiguous")


def _scales(k_scale, v_scale):
    return (k_scale.data_ptr(), *k_scale.stride(), v_scale.data_ptr(), *v_scale.stride())


def alloc_kv_scales(num_blocks: int, hkv: int, device) -> Tuple[torch.Tensor, torch.Tensor]:
    """Scales of a cache, ones: keys and values of a (block, head) side by side, since attention reads them together."""
    both = torch.ones(num_blocks, hkv, 2, dtype=torch.float32, device=device)
    return both[..., 0], both[..., 1]


def qk_norm_rope_kv_write(q, k, v, positions, rope_cache, rotary_dim, k_cache, v_cache, slot_mapping, k_scale, v_scale, q_norm_w=None,
                          k_norm_w=None, eps=1e-6, norm_plus_one=False, norm_dim=0) -> torch.Tensor:
    nb, hkv, d = check_cache(k_cache, v_cache, k_scale, v_scale)
    _writable(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.get_device()
    for x, what in ((q, "queries"), (k, "keys"), (v, "values")):
        _heads(x, what, dev, d)
    T, hq, _ = q.shape
    if k.shape[0] != T or v.shape[0] != T or k.shape[1] != hkv or v.shape[1] != hkv:
        raise K.KernelError(f"{T} rows of queries and {hkv} heads of the cache beside keys {tuple(k.shape)} and values {tuple(v.shape)}")
    _ints(slot_mapping, "slots", dev, 1)
    if slot_mapping.shape[0] != T:
        raise K.KernelError(f"{slot_mapping.shape[0]} slots for {T} rows")
    pos = rope = 0
    if rotary_dim:
        _ints(positions, "positions", dev, 1)
        if rotary_dim < 0 or rotary_dim > d or rotary_dim % 16:
            raise K.KernelError(f"the rotated width of {d}-wide heads is a multiple of 16, at most {d}, not {rotary_dim}")
        if positions.shape[0] != T or rope_cache.dtype != _F32 or rope_cache.dim() != 2 or rope_cache.shape[1] != rotary_dim \
                or not rope_cache.is_contiguous() or rope_cache.get_device() != dev:
            raise K.KernelError("rotation: a position per row and an fp32 [positions, rotary_dim] table beside the cache")
        pos, rope = positions.data_ptr(), rope_cache.data_ptr()
    if (q_norm_w is None) != (k_norm_w is None):
        raise K.KernelError("head norms come for queries and keys together")
    qw = kw = 0
    if q_norm_w is not None:
        for w in (q_norm_w, k_norm_w):
            if w.dtype != _BF16 or w.shape != (d,) or not w.is_contiguous() or w.get_device() != dev:
                raise K.KernelError(f"head norm weights are bf16 [{d}]")
        qw, kw = q_norm_w.data_ptr(), k_norm_w.data_ptr()
    if T == 0:
        return torch.empty_like(q)
    if checked.ENABLED:
        checked.kv_write(slot_mapping, positions, nb, BLOCK, rope_cache.shape[0] if rotary_dim else 0)
        checked.block_runs(slot_mapping, BLOCK)
    guard, _, stream = _place(k_cache)
    with guard:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        _call("atlas_kv_scaled_write", _WRITE.pack(
            q.data_ptr(), q.stride(0), out.data_ptr(), hq * d, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), pos, rope, qw, kw,
            k_cache.data_ptr(), v_cache.data_ptr(), *_scales(k_scale, v_scale), slot_mapping.data_ptr(), T, hq, hkv, d, rotary_dim, nb,
            1 if norm_plus_one else 0, norm_dim or d, eps, stream), "kv_scaled_write")
    return out


def kv_read(k_cache, v_cache, block_tables, seq_lens, max_len: int, k_scale, v_scale) -> Tuple[torch.Tensor, torch.Tensor]:
    nb, hkv, d = check_cache(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.get_device()
    _ints(block_tables, "block tables", dev, 2)
    _ints(seq_lens, "sequence lengths", dev, 1)
    B, cols = block_tables.shape
    if seq_lens.shape[0] != B or max_len < 0:
        raise K.KernelError(f"{seq_lens.shape[0]} lengths for {B} block tables, {max_len} tokens of each")
    out = torch.empty((2, B, max_len, hkv, d), dtype=_BF16, device=k_cache.device)
    if out.numel():
        guard, _, stream = _place(k_cache)
        at = out.data_ptr()
        with guard:
            _call("atlas_kv_scaled_read", _READ.pack(
                k_cache.data_ptr(), v_cache.data_ptr(), *_scales(k_scale, v_scale), block_tables.data_ptr(), block_tables.stride(0), cols,
                seq_lens.data_ptr(), B, max_len, hkv, d, nb, at, at + B * max_len * hkv * d * 2, stream), "kv_scaled_read")
    return out.unbind(0)


def kv_evict(k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens, weights, keep: int, new_tables, sink: int, recent: int):
    nb, hkv, d = check_cache(k_cache, v_cache, k_scale, v_scale)
    _writable(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.get_device()
    for t, what, n in ((block_tables, "block tables", 2), (new_tables, "new block tables", 2), (seq_lens, "sequence lengths", 1)):
        _ints(t, what, dev, n)
    B, cols = block_tables.shape
    if keep < 1 or sink < 0 or recent < 0 or sink + recent > keep:
        raise K.KernelError(f"keeping {keep} tokens of which the first {sink} and the last {recent} are fixed")
    if weights.dtype != _F32 or weights.dim() != 3 or weights.shape[:2] != (B, hkv) or weights.get_device() != dev \
            or (weights.numel() and weights.stride(2) != 1):
        raise K.KernelError(f"weights are fp32 [{B}, {hkv}, tokens] beside the cache, tokens contiguous")
    width = min(weights.shape[2], cols * BLOCK)                        # no sequence is longer
    need = (min(keep, width) + BLOCK - 1) // BLOCK
    if seq_lens.shape[0] != B or new_tables.shape[0] != B or new_tables.shape[1] < need:
        raise K.KernelError(f"{B} sequences that keep up to {min(keep, width)} tokens need their lengths and new block tables of {need} columns")
    kept = torch.empty((B, hkv, keep), dtype=_I32, device=k_cache.device)
    out_w = torch.empty((B, hkv, keep), dtype=_F32, device=k_cache.device)
    lens = torch.empty(B, dtype=_I32, device=k_cache.device)
    if B == 0:
        return lens, kept, out_w
    if checked.ENABLED:
        checked.evict(block_tables, seq_lens, new_tables, nb, BLOCK, keep, width)
    guard, index, stream = _place(k_cache)
    with guard:
        _call("atlas_kv_evict", _EVICT.pack(
            k_cache.data_ptr(), v_cache.data_ptr(), *_scales(k_scale, v_scale), block_tables.data_ptr(), block_tables.stride(0),
            seq_lens.data_ptr(), weights.data_ptr(), weights.stride(0), weights.stride(1), width, B, hkv, d, nb, keep, sink, recent,
            new_tables.data_ptr(), new_tables.stride(0), lens.data_ptr(), kept.data_ptr(), out_w.data_ptr(), K._num_sms[index], stream), "kv_evict")
    return lens, kept, out_w


def _weigh_tiles(batch, nd: int, device):
    """Tiles of 128 cached tokens of the chunk sequences, those with the most rows first: (device [2, n], n)."""
    def build():
        work = []
        for i in range(nd, batch.num_seqs):
            n, rows = batch.seq_lens_host[i], batch.query_lens_host[i]
            if rows:
                work += [(-(rows - max(0, k0 - (n - rows))), i, k0) for k0 in range(0, n, 128)]
        work.sort()
        return [w[1] for w in work], [w[2] for w in work]
    return K.step_list(batch, "cached", build, device)


def key_shares(lens, items: int, window: int, sms: int) -> int:
    """Shares of the keys of prompt rows' sequences of ``lens`` tokens.  Few query tiles behind many keys: as many as fill the GPU once, at least
    512 tokens of the longest each."""
    longest = max(lens, default=0)
    return max(1, min(sms // items, (min(longest, window + 128) if window else longest) // 512)) if items else 1


def paged_attention(q, k_cache, v_cache, batch, scale, k_scale, v_scale, sliding_window: Optional[int] = None,
                    weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    nb, hkv, d = check_cache(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.get_device()
    _heads(q, "queries", dev, d)
    T, hq, _ = q.shape
    g = hq // hkv
    if hq % hkv or not 1 <= g <= 128:
        raise K.KernelError(f"{hq} query heads over {hkv} key heads: 1 to 128 for each")
    ldq, at_q = q.stride(0), q.data_ptr()
    if ldq % 8 or at_q % 16:
        raise K.KernelError("queries start on 16 bytes in every row")
    bt, lens, starts = batch.block_tables, batch.seq_lens, batch.query_start_loc
    _ints(bt, "block tables", dev, 2)
    _ints(lens, "sequence lengths", dev, 1)
    _ints(starts, "query starts", dev, 1)
    window, nd, B = int(sliding_window or 0), batch.num_decodes, lens.shape[0]
    rows, cols = bt.shape
    longest = batch.max_seq_len
    window = min(window, max(1, cols * BLOCK))              # no sequence is longer: the kernels' sums of positions stay in 32 bits
    if window < 0 or rows < B or starts.shape[0] < B + 1 or not 0 <= nd <= B or T < nd:
        raise K.KernelError("attention: a block table, a length and a start for every sequence, a row for every decode, no negative window")
    if B > nd and (len(batch.query_lens_host) < B or len(batch.seq_lens_host) < B or nd + sum(batch.query_lens_host[nd:B]) > T):
        raise K.KernelError(f"{T} query rows for {nd} single tokens and chunks of {list(batch.query_lens_host[nd:B])}, whose host lengths a batch has")
    if not 2.0 ** -60 <= scale <= 2.0 ** 60:              # scores are masked, and the largest is taken, before it is applied
        raise K.KernelError(f"the softmax scale is positive, from 2^-60 to 2^60, not {scale}")
    width, sums = 0, (0, 0, 0)
    if weights is not None:
        if weights.dtype != _F32 or weights.dim() != 3 or weights.shape[:2] != (B, hkv) or weights.get_device() != dev \
                or weights.stride(2) != 1 or weights.shape[2] < longest:
            raise K.KernelError(f"weights are fp32 [{B}, {hkv}, at least {longest}] beside the cache, tokens contiguous")
        if not (weights.is_contiguous() or _apart(weights)):
            raise K.KernelError("weights: every sequence and head has sums of its own")
        width = weights.shape[2]
        sums = (weights.data_ptr(), weights.stride(0), weights.stride(1))
    if T == 0 or B == 0:
        return torch.empty_like(q)
    if checked.ENABLED:
        checked.paged_read(bt, lens, nb, BLOCK)
    guard, index, stream = _place(k_cache)
    with guard:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        cache = (k_cache.data_ptr(), v_cache.data_ptr(), *_scales(k_scale, v_scale), bt.data_ptr(), bt.stride(0), cols, lens.data_ptr(),
                 starts.data_ptr())
        status, at_out = K._status_ptr[index], out.data_ptr()
        if nd > 0:
            n_cols, items = min((g + 1) // 2 * 2, 16), nd * hkv * ((g + 15) // 16)
            pages = items * ((longest + BLOCK - 1) // BLOCK)
            blocks = max(1, min((pages + LEAST - 1) // LEAST, K._num_sms[index]))
            pieces = items + blocks * WARPS
            n_o, n_ml = pieces * n_cols * d, pieces * n_cols * 2
            n_s = n_r = tokens = 0
            if weights is not None:
                # the scores go through memory, for as many tokens as there are; a graph's sequences grow up to the width of the sums
                tokens = width if longest <= 0 or torch._C._cuda_isCurrentStreamCapturing() else min(width, longest)
                n_s, n_r = nd * hkv * tokens * ((g + 1) // 2 * 2), nd * hq * 2
            work = torch.empty(n_o + n_ml + n_s + n_r, dtype=_F32, device=q.device)       # every part a multiple of 16 bytes or the last
            at = work.data_ptr()
            at_s = at + 4 * (n_o + n_ml)
            _call("atlas_attn_scaled_decode", _DECODE.pack(
                at_q, ldq, at_out, hq * d, *cache, nd, hq, hkv, d, window, nb, longest, blocks, at, at + 4 * n_o, at_s if n_s else 0, tokens,
                at_s + 4 * n_s if n_r else 0, *sums, scale, status, stream), "attn_scaled_decode")
        if B > nd:
            tiles, n, _ = K._tc_tiles(q, batch, nd, 128 // g * (2 if d <= 128 else 1))
            ml = key_tiles = parts = None
            at_keys = n_keys = n_o = 0
            splits = key_shares(batch.seq_lens_host[nd:], n * hkv, window, K._num_sms[index])
            if splits > 1:
                n_o = splits * (T - nd) * hq * d
                parts = torch.empty(n_o + splits * (T - nd) * hq * 2, dtype=_F32, device=q.device)
            if weights is not None:
                ml = torch.empty((T, hq, 2), dtype=_F32, device=q.device)
                key_tiles, n_keys = _weigh_tiles(batch, nd, q.device)
                at_keys = key_tiles.data_ptr()
            at = tiles.data_ptr()
            _call("atlas_attn_scaled_chunk", _CHUNK.pack(
                at_q, ldq, at_out, hq * d, *cache, at, at + 4 * n, n, T, hq, hkv, d, window, nb, 0 if ml is None else ml.data_ptr(), splits, nd,
                parts.data_ptr() if n_o else 0, parts.data_ptr() + 4 * n_o if n_o else 0, at_keys,
                at_keys + 4 * n_keys, n_keys, *sums, width, K._num_sms[index], scale, status, stream), "attn_scaled_chunk")
    return out

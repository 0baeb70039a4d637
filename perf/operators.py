"""The operators of an 8-bit paged cache whose scales go by block: writing it, attending over it, counting which tokens attention
looks at, and keeping only those.

A block of 16 tokens of one head holds ``e4m3`` numbers and one power of two.  With ``a`` the largest magnitude among a block's
tokens, its scale is the smallest ``2^e`` (``-60 <= e <= 60``) with ``a <= 448 * 2^e``, and a token holds ``round(x / 2^e)``.
Appending to a block never lowers its scale; where it raises it, the tokens that are there move over by the quotient of the two.

=========  =============================================================================================================
op         one pass
=========  =============================================================================================================
write      RMS norm of the heads (some models), rotation, block scales, rounding, cache write; the rotated queries and the
           written blocks' values come back
attend     attention of a step's rows over the cache: ``dec`` sequences with one new token, then ``chunks`` with ``rows``
weigh      the same, and every cached token's softmax weight, summed over the step's rows and a key head's query heads,
           joins the running sums ``weights [sequence, key head, token]``
evict      per sequence and key head the first ``sink`` tokens, the last ``recent`` and, of those between, the heaviest
           move to new blocks in their order until ``keep`` are there; ties go to the earlier token
=========  =============================================================================================================

Sizes: ``hkv`` key heads with ``g`` query heads each, ``d`` wide; ``ctx`` tokens are in the cache of a chunk before its rows; decode
sequences hold ``len`` tokens with the new one; with ``ragged`` these are the largest and the others fall off to a quarter.
"""
import math

import torch

own = False
PAGE = 16
LOW, HIGH = -60, 60


def listed():
    return [
        # appending one token each for a full server: every row lands inside a block that others have begun
        dict(name="write-decode-128", op="write", hkv=8, g=4, d=128, rot=128, norm=False, seqs=128, rows=1, ctx=1151, ragged=True),
        # a full prefill step of eight prompts
        dict(name="write-prompt-8x1024", op="write", hkv=8, g=4, d=128, rot=128, norm=False, seqs=8, rows=1024, ctx=0, ragged=False),
        # wide heads with head norms and a quarter rotated, the rest of a prompt behind a cached prefix that ends inside a block
        dict(name="write-rest-517+4099", op="write", hkv=2, g=8, d=256, rot=64, norm=True, seqs=1, rows=517, ctx=4099, ragged=False),
        # one user's short chat: latency
        dict(name="decode-1x77", op="attend", hkv=8, g=4, d=128, dec=1, len=77, chunks=0, rows=0, ctx=0, ragged=False, window=0),
        # a full server at the headline workload's lengths
        dict(name="decode-128x1152", op="attend", hkv=8, g=4, d=128, dec=128, len=1152, chunks=0, rows=0, ctx=0, ragged=False, window=0),
        # three users of wide heads, one of them far into a long document
        dict(name="decode-3x65531", op="attend", hkv=2, g=8, d=256, dec=3, len=65531, chunks=0, rows=0, ctx=0, ragged=True, window=0),
        # a prefill step, and the rest of a prompt behind 4096 tokens beside running decodes
        dict(name="prompt-8x1024", op="attend", hkv=8, g=4, d=128, dec=0, len=0, chunks=8, rows=1024, ctx=0, ragged=False, window=0),
        dict(name="mixed-37+517+4096", op="attend", hkv=2, g=8, d=256, dec=37, len=2999, chunks=1, rows=517, ctx=4096, ragged=True, window=0),
        # decode steps of a server that will evict: ordinary contexts
        dict(name="weigh-decode-32x4096", op="weigh", hkv=8, g=4, d=128, dec=32, len=4096, chunks=0, rows=0, ctx=0, ragged=True, window=0),
        # the prompt's own rows say which of its tokens matter
        dict(name="weigh-prompt-2x3001", op="weigh", hkv=8, g=4, d=128, dec=0, len=0, chunks=2, rows=3001, ctx=0, ragged=True, window=0),
        # a server's caches cut to a quarter, and one long document to 4096 tokens
        dict(name="evict-32x4096", op="evict", hkv=8, g=4, d=128, seqs=32, len=4096, ragged=True, keep=1024, sink=4, recent=64),
        dict(name="evict-1x65531", op="evict", hkv=8, g=4, d=128, seqs=1, len=65531, ragged=False, keep=4096, sink=16, recent=512),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Lengths from one token on, one sequence to many, every head width, groups of one to sixteen query heads."""
    op = rng.choice(["write", "attend", "attend", "attend", "weigh", "weigh", "evict"])
    d = rng.choice([64, 128, 128, 128, 256])
    hkv = rng.choice([1, 2, 2, 4, 5, 8])
    g = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
    case = dict(op=op, hkv=hkv, g=g, d=d, ragged=rng.random() < 0.6)
    room = 8 * 128 * 4 / (hkv * g * d)                                    # query widths against those of the listed cases
    if op == "write":
        case.update(rot=rng.choice([d, d // 2, d // 4]), norm=rng.random() < 0.5, ctx=rng.choice([0, _log(rng, 1, 8000)]))
        case["seqs"] = _log(rng, 1, 100)
        case["rows"] = 1 if rng.random() < 0.3 else _log(rng, 1, max(2, min(4000, 8000 * room / case["seqs"])))
    elif op == "evict":
        case["seqs"] = _log(rng, 1, 24)
        case["len"] = _log(rng, 40, min(65000, 400000 / (case["seqs"] * hkv * d / 256)))
        case["keep"] = max(24, _log(rng, 24, max(25, case["len"])))
        case["sink"], case["recent"] = rng.choice([0, 1, 4, 16]), rng.choice([0, 1, 8])
    else:
        case.update(dec=0, len=0, chunks=0, rows=0, ctx=0, window=rng.choice([0, 0, 0, _log(rng, 1, 3000)]))
        kind = rng.choice(["dec", "dec", "chunk", "chunk", "both"])
        if kind != "chunk":
            case["dec"] = _log(rng, 1, 128)
            case["len"] = _log(rng, 1, max(2, min(65000, (550000 if kind == "dec" else 200000) / (case["dec"] * hkv * d / 256))))
        if kind != "dec":
            case["chunks"] = _log(rng, 1, 8)
            case["rows"] = _log(rng, 2, max(3, min(2000, 4000 * room / case["chunks"])))
            case["ctx"] = rng.choice([0, _log(rng, 1, max(2, min(5000, 2e6 * room / (case["chunks"] * case["rows"]))))])
    return case


# ----------------------------------------------------------------------------- sizes of a case
def _fall(n, i, ragged):
    return max(1, int(n * (1.0 - 0.75 * ((i * 37) % 101) / 100.0))) if ragged else max(1, n)


def _lens(case):
    """(tokens in the cache after the step, new rows) per sequence; decodes first."""
    if case["op"] == "write":
        rows = [_fall(case["rows"], i, case["ragged"] and case["rows"] > 1) for i in range(case["seqs"])]
        ctx = [_fall(case["ctx"], i, case["ragged"]) if case["ctx"] else 0 for i in range(case["seqs"])]
        return [c + r for c, r in zip(ctx, rows)], rows
    if case["op"] == "evict":
        return [_fall(case["len"], i, case["ragged"]) for i in range(case["seqs"])], [0] * case["seqs"]
    lens = [_fall(case["len"], i, case["ragged"]) for i in range(case["dec"])]
    rows = [1] * case["dec"]
    for i in range(case["chunks"]):
        r = max(2, _fall(case["rows"], i, case["ragged"]))
        rows.append(r)
        lens.append(r + (_fall(case["ctx"], i, case["ragged"]) if case["ctx"] else 0))
    return lens, rows


def _pairs(lens, rows, window):
    """(query, key) pairs that the masks leave, and keys that some row sees."""
    pairs = keys = 0
    for n, r in zip(lens, rows):
        lo = n - r                                                        # position of the first row
        w = window or n
        if lo + 1 >= w:
            pairs += r * w
        else:
            grow = min(r, w - lo - 1)                                     # rows whose window still reaches the start
            pairs += grow * (lo + 1) + grow * (grow - 1) // 2 + (r - grow) * w
        keys += min(n, w + r - 1)
    return pairs, keys


def work(case):
    hkv, g, d = case["hkv"], case["g"], case["d"]
    lens, rows = _lens(case)
    new = sum(rows)
    if case["op"] == "write":
        pages = sum((n + PAGE - 1) // PAGE - (n - r) // PAGE for n, r in zip(lens, rows))
        cells = new + sum((n - r) % PAGE for n, r in zip(lens, rows))
        return {"bytes": 4 * new * hkv * g * d + 4 * new * hkv * d + 2 * new * hkv * d + 4 * new * case["rot"]
                         + 2 * cells * hkv * d * 3 + 8 * pages * hkv,
                "flops": 10 * new * (hkv * g + 2 * hkv) * d}
    if case["op"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lens)
        return {"bytes": 4 * sum(lens) * hkv + 8 * kept * hkv + 4 * kept * hkv * d + 4 * kept * hkv * d + 2 * kept * hkv * d,
                "flops": 4 * kept * hkv * d}
    pairs, keys = _pairs(lens, rows, case["window"])
    size = 2 * keys * hkv * d + 8 * (keys // PAGE + 1) * hkv + 4 * new * hkv * g * d
    flops = 4 * pairs * hkv * g * d
    if case["op"] == "weigh":
        size += 8 * sum(lens) * hkv
        if case["chunks"]:                            # the rows' sums come first: the scores are formed twice
            at = slice(case["dec"], None)
            flops += 2 * _pairs(lens[at], rows[at], case["window"])[0] * hkv * g * d
    return {"bytes": size, "flops": flops}


# ----------------------------------------------------------------------------- inputs
def _pow2(x):
    return torch.ldexp(torch.ones_like(x, dtype=torch.float32), x.to(torch.int32))


def _exponent(a):
    """Smallest e in [-60, 60] with a <= 448 * 2^e (fp32 magnitudes)."""
    m, x = torch.frexp(a)                                                 # a = m 2^x with m in [1/2, 1); 448 = 7/8 2^9
    e = torch.where(m <= 0.875, x - 9, x - 8)
    return torch.where(a > 0, e, torch.full_like(e, LOW)).clamp(LOW, HIGH)


def _quantised(x):
    """``x [blocks, heads, 16, d]`` (fp32) -> bytes and scales of a cache."""
    e = _exponent(x.abs().amax((2, 3)))
    s = _pow2(e)
    return (x / s[:, :, None, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), s


def _pool(case, blocks, gen):
    """A filled cache.  Keys have a few loud channels, as trained models have them; blocks differ in loudness."""
    hkv, d = case["hkv"], case["d"]
    dev = torch.device("cuda")
    loud = 1.0 + 5.0 * (torch.rand(hkv, 1, d, generator=gen, device=dev) < 0.04).float()
    out = []
    for values in (False, True):
        cells, scales = [], []
        for lo in range(0, blocks, 8192):
            n = min(8192, blocks - lo)
            x = torch.randn(n, hkv, PAGE, d, generator=gen, device=dev)
            x *= torch.exp(0.7 * torch.randn(n, hkv, 1, 1, generator=gen, device=dev)) if values else loud
            c, s = _quantised(x)
            cells.append(c)
            scales.append(s)
        raw = torch.cat([c.view(torch.uint8) for c in cells]).view(torch.float8_e4m3fn)
        out.append((raw, torch.cat(scales)))
    (k, ks), (v, vs) = out
    v = v.view(torch.uint8).transpose(2, 3).contiguous().view(torch.float8_e4m3fn)    # a value block lies token by token in a row
    return k, v, ks, vs


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    hkv, g, d = case["hkv"], case["g"], case["d"]
    lens, rows = _lens(case)
    n_pages = [(n + PAGE - 1) // PAGE for n in lens]
    blocks = sum(n_pages) + 3
    state = dict(case=case, lens=lens, rows=rows)
    k, v, ks, vs = _pool(case, blocks, gen)
    state.update(k_raw=k, v_raw=v, k=k.permute(0, 2, 1, 3), v=v.permute(0, 3, 1, 2), ks=ks, vs=vs)
    order = torch.randperm(blocks, generator=gen, device=dev).to(torch.int32)
    starts = [sum(n_pages[:i]) for i in range(len(lens))]
    wide = max(n_pages)
    at = torch.tensor(starts, device=dev)[:, None] + torch.arange(wide, device=dev)[None]
    live = torch.arange(wide, device=dev)[None] < torch.tensor(n_pages, device=dev)[:, None]
    state["tables"] = torch.where(live, order[at.clamp(max=blocks - 1)], torch.zeros((), dtype=torch.int32, device=dev))
    state["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    new = sum(rows)
    ends = torch.tensor(rows).cumsum(0).tolist()
    state["starts"] = torch.tensor([0] + ends, dtype=torch.int32, device=dev)
    if case["op"] == "write":
        qkv = torch.randn(new, (g + 2) * hkv * d, generator=gen, device=dev)
        loud = 1.0 + 5.0 * (torch.rand(hkv * d, generator=gen, device=dev) < 0.04).float()
        qkv[:, g * hkv * d:(g + 1) * hkv * d] *= loud
        qkv[:, (g + 1) * hkv * d:] *= torch.exp(0.7 * torch.randn(new, 1, generator=gen, device=dev))
        qkv = qkv.to(torch.bfloat16)
        state["q"] = qkv[:, :g * hkv * d].view(new, g * hkv, d)
        state["key"] = qkv[:, g * hkv * d:(g + 1) * hkv * d].view(new, hkv, d)
        state["value"] = qkv[:, (g + 1) * hkv * d:].view(new, hkv, d)
        seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(rows)).to(dev)
        pos = torch.cat([torch.arange(n - r, n) for n, r in zip(lens, rows)]).to(dev)
        state["positions"] = pos.to(torch.int32)
        state["slots"] = (state["tables"][seq, pos // PAGE] * PAGE + pos % PAGE).to(torch.int32)
        turn = torch.outer(torch.arange(max(lens), dtype=torch.float64, device=dev),
                           5e5 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device=dev) / case["rot"]))
        state["rope"] = torch.cat([turn.cos(), turn.sin()], 1).float()
        state["norms"] = [(1.0 + 0.2 * torch.randn(d, generator=gen, device=dev)).to(torch.bfloat16) for _ in range(2)] if case["norm"] else [None, None]
        # the written blocks: where they are, how many tokens they held, how many they hold now
        first = [(n - r) // PAGE for n, r in zip(lens, rows)]
        touched = [(i, p) for i in range(len(lens)) for p in range(first[i], n_pages[i])]
        ti, tp = torch.tensor(touched).t().to(dev)
        state["touched"] = state["tables"][ti, tp][:, None].contiguous()
        held = torch.tensor([max(0, lens[i] - rows[i] - p * PAGE) for i, p in touched])
        holds = torch.tensor([min(PAGE, lens[i] - p * PAGE) for i, p in touched])
        state["held"], state["holds"] = held.to(dev), holds.to(torch.int32).to(dev)
        base = torch.tensor([0] + [n_pages[i] - first[i] for i in range(len(lens))]).cumsum(0)[:-1].to(dev)
        state["page_of_row"] = base[seq] + pos // PAGE - torch.tensor(first, device=dev)[seq]
    elif case["op"] == "evict":
        spread = torch.randn(len(lens), hkv, max(lens), generator=gen, device=dev)
        state["weights"] = torch.exp(2.0 * spread) * (torch.rand(spread.shape, generator=gen, device=dev) > 0.2)   # many were never looked at
        kept_pages = [(min(n, case["keep"]) + PAGE - 1) // PAGE for n in lens]
        spare = sum(kept_pages)
        for name, raw in (("k", k), ("v", v)):                            # blocks for what is kept, behind the pool
            grown = torch.cat([raw.view(torch.uint8), torch.zeros((spare,) + tuple(raw.shape[1:]), dtype=torch.uint8, device=dev)]).view(raw.dtype)
            state[name + "_raw"] = grown
            state[name] = grown.permute(0, 2, 1, 3) if name == "k" else grown.permute(0, 3, 1, 2)
        one = torch.ones(spare, hkv, device=dev)
        state["ks"], state["vs"] = torch.cat([ks, one]), torch.cat([vs, one])
        to = torch.zeros(len(lens), max(kept_pages), dtype=torch.int32)
        at, ids = 0, (blocks + torch.randperm(spare, generator=gen, device=dev)).to(torch.int32).cpu()
        for i, n in enumerate(kept_pages):
            to[i, :n] = ids[at:at + n]
            at += n
        state["to"] = to.to(dev)
    else:
        loud = 1.0 + 2.0 * (torch.rand(hkv * g, 1, generator=gen, device=dev) < 0.3).float()       # some heads look sharply
        state["q"] = (torch.randn(new, hkv * g, d, generator=gen, device=dev) * 0.5 * loud).to(torch.bfloat16)
        if case["op"] == "weigh":
            state["weights"] = 3.0 * torch.rand(len(lens), hkv, max(lens), generator=gen, device=dev)
        if own:
            state["batch"] = _step(state)
    return state


def _step(state):
    """The step's metadata as an engine keeps it."""
    from atlas_b200.models.batch import ForwardBatch
    case, lens, rows = state["case"], state["lens"], state["rows"]
    new = sum(rows)
    dev = state["q"].device
    pos = torch.cat([torch.arange(n - r, n) for n, r in zip(lens, rows)]).to(torch.int32).to(dev)
    return ForwardBatch(input_ids=torch.zeros(new, dtype=torch.int64, device=dev), positions=pos,
                        slot_mapping=torch.full((new,), -1, dtype=torch.int32, device=dev), block_tables=state["tables"],
                        seq_lens=state["seq_lens"], query_start_loc=state["starts"], num_decodes=case["dec"], max_query_len=max(rows),
                        max_seq_len=max(lens), seq_lens_host=lens, query_lens_host=rows)


def run(state):
    case = state["case"]
    return {"write": _write, "evict": _evict}.get(case["op"], _attend)(state, case)


# ----------------------------------------------------------------------------- plain forms
def _read(cells, scales, tables):
    """fp32 values of the blocks ``tables [n, p]`` of a cache ``[blocks, heads, 16, d]``: ``[n, heads, p * 16, d]``."""
    n, p = tables.shape
    at = tables.reshape(-1).long()
    x = cells.view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * scales[at][:, :, None, None]
    h, d = x.shape[1], x.shape[3]
    return x.view(n, p, h, PAGE, d).transpose(1, 2).reshape(n, h, p * PAGE, d)


def _rounded(x, scales):
    return (x / scales[:, :, None, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _turn(x, norm, state):
    x = x.float()
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * norm.float()
    half = state["case"]["rot"] // 2
    cs = state["rope"][state["positions"].long()][:, None]
    c, s = cs[..., :half], cs[..., half:]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:]], -1)


def _write(state, case):
    if own:
        from atlas_b200 import ops
        q = ops.qk_norm_rope_kv_write(state["q"], state["key"], state["value"], state["positions"], state["rope"], case["rot"], state["k"],
                                      state["v"], state["slots"], state["ks"], state["vs"], *state["norms"])
        return (q,) + ops.kv_read(state["k"], state["v"], state["touched"], state["holds"], PAGE, state["ks"], state["vs"])
    q = _turn(state["q"], state["norms"][0], state)
    blocks, of_row = state["touched"][:, 0].long(), state["page_of_row"]
    off = state["slots"].long() % PAGE
    held, holds = state["held"][:, None], state["holds"][:, None]
    token = torch.arange(PAGE, device=off.device)[None]
    out = [q.to(torch.bfloat16)]
    for x, cells, scales in ((_turn(state["key"], state["norms"][1], state), state["k_raw"], state["ks"]),
                             (state["value"].float(), state["v_raw"], state["vs"])):
        byte = cells.view(torch.uint8)
        flat = byte if cells is state["k_raw"] else byte.transpose(2, 3)
        was = flat[blocks].view(torch.float8_e4m3fn).float()                        # [n, heads, 16, d]
        largest = torch.zeros(blocks.shape[0], x.shape[1], device=x.device).index_reduce_(0, of_row, x.abs().amax(-1), "amax")
        before = scales[blocks]
        scale = torch.where(held > 0, torch.maximum(_pow2(_exponent(largest)), before), _pow2(_exponent(largest)))
        now = torch.where((token < held)[:, None, :, None], was * (before / scale)[:, :, None, None], torch.zeros_like(was))
        now = now.transpose(1, 2).contiguous()
        now[of_row, off] = x / scale[of_row][:, :, None]
        now = now.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).transpose(1, 2)     # [n, heads, 16, d]
        live = (token < holds)[:, None, :, None]
        flat[blocks] = torch.where(live, now.view(torch.uint8), flat[blocks])
        scales[blocks] = scale
        out.append(torch.where(live, now.float() * scale[:, :, None, None], torch.zeros((), device=x.device)).transpose(1, 2).to(torch.bfloat16))
    return tuple(out)


def _attend(state, case):
    weights = state["weights"].clone() if case["op"] == "weigh" else None
    scale = case["d"] ** -0.5
    if own:
        from atlas_b200 import ops
        out = ops.paged_attention(state["q"], state["k"], state["v"], state["batch"], scale, state["ks"], state["vs"], case["window"] or None,
                                  weights=weights)
        return out if weights is None else (out, weights)
    hkv, g, d = case["hkv"], case["g"], case["d"]
    v_cells = state["v_raw"].transpose(2, 3)
    out = torch.zeros_like(state["q"])
    lens, rows, dec = state["lens"], state["rows"], case["dec"]

    def some(q, k, v, hi):
        """``q [n, heads, g, r, d]``, keys up to ``hi [n, r]``; returns the output and the rows' weights' sums."""
        s = (q @ k.transpose(-1, -2)[:, :, None]) * scale
        j = torch.arange(k.shape[2], device=q.device)
        dead = j > hi[..., None]
        if case["window"]:
            dead |= j <= hi[..., None] - case["window"]
        s = s.masked_fill(dead[:, None, None], float("-inf"))
        e = torch.exp(s - s.amax(-1, keepdim=True))
        p = e / e.sum(-1, keepdim=True)
        return p @ v[:, :, None], p.sum((2, 3)) if weights is not None else None

    step = max(1, int(2e9 // (max(lens) * hkv * max(d, g) * 4)))
    for lo in range(0, dec, step):
        n = min(step, dec - lo)
        wide = (max(lens[lo:lo + n]) + PAGE - 1) // PAGE
        tab = state["tables"][lo:lo + n, :wide]
        k, v = _read(state["k_raw"], state["ks"], tab), _read(v_cells, state["vs"], tab)
        q = state["q"][lo:lo + n].float().view(n, hkv, g, 1, d)
        o, w = some(q, k, v, state["seq_lens"][lo:lo + n, None].long() - 1)
        out[lo:lo + n] = o.reshape(n, hkv * g, d).to(out.dtype)
        if weights is not None:
            most = min(w.shape[2], weights.shape[2])
            weights[lo:lo + n, :, :most] += w[:, :, :most]
    row = dec
    for i in range(dec, len(lens)):
        n, r = lens[i], rows[i]
        tab = state["tables"][i:i + 1, :(n + PAGE - 1) // PAGE]
        k, v = _read(state["k_raw"], state["ks"], tab)[:, :, :n], _read(v_cells, state["vs"], tab)[:, :, :n]
        step = max(1, int(1.5e9 // (n * hkv * g * 4)))
        for lo in range(0, r, step):
            m = min(step, r - lo)
            q = state["q"][row + lo:row + lo + m].float().view(m, hkv, g, d).permute(1, 2, 0, 3)[None]
            hi = n - r + lo + torch.arange(m, device=q.device)[None]
            o, w = some(q, k, v, hi)
            out[row + lo:row + lo + m] = o[0].permute(2, 0, 1, 3).reshape(m, hkv * g, d).to(out.dtype)
            if weights is not None:
                weights[i, :, :n] += w[0]
        row += r
    return out if weights is None else (out, weights)


def _evict(state, case):
    if own:
        from atlas_b200 import ops
        lens, kept, weights = ops.kv_evict(state["k"], state["v"], state["ks"], state["vs"], state["tables"], state["seq_lens"], state["weights"],
                                           case["keep"], state["to"], sink=case["sink"], recent=case["recent"])
        return (lens, kept, weights) + ops.kv_read(state["k"], state["v"], state["to"], lens, case["keep"], state["ks"], state["vs"])
    hkv, keep = case["hkv"], case["keep"]
    weights = state["weights"]
    length = state["seq_lens"].long()[:, None, None]
    j = torch.arange(weights.shape[2], device=weights.device)[None, None]
    rank = torch.where((j < case["sink"]) | (j >= length - case["recent"]), torch.full_like(weights, float("inf")), weights)
    rank = torch.where(j < length, rank, torch.full_like(rank, float("-inf")))
    order = torch.sort(rank, dim=2, descending=True, stable=True).indices[:, :, :keep]
    if order.shape[2] < keep:
        order = torch.cat([order, order.new_full(order.shape[:2] + (keep - order.shape[2],), weights.shape[2])], 2)
    lens = length[:, 0, 0].clamp(max=keep)
    slot = torch.arange(keep, device=weights.device)[None, None]
    order = torch.where(slot < lens[:, None, None], order, torch.full_like(order, 1 << 30))
    kept = torch.sort(order, dim=2).values
    live = slot < lens[:, None, None]
    at = torch.where(live, kept, torch.zeros_like(kept))
    out_w = torch.where(live, weights.gather(2, at), torch.zeros((), device=weights.device))
    n, p = state["to"].shape
    result = [lens.to(torch.int32), torch.where(live, kept, torch.full_like(kept, -1)).to(torch.int32), out_w]
    block = state["tables"].long().gather(1, (at // PAGE).view(n, -1)).view(at.shape)
    head = torch.arange(hkv, device=at.device)[None, :, None]
    pad = p * PAGE - keep
    to, used = state["to"].long(), torch.arange(p, device=at.device)[None] * PAGE < lens[:, None]
    for cells, scales in ((state["k_raw"], state["ks"]), (state["v_raw"].transpose(2, 3), state["vs"])):
        x = cells.view(torch.uint8)[block, head, at % PAGE].view(torch.float8_e4m3fn).float() * scales[block, head][..., None]
        x = torch.where(live[..., None], x, torch.zeros((), device=x.device))             # [n, heads, keep, d]
        x = torch.nn.functional.pad(x, (0, 0, 0, pad)) if pad >= 0 else x[:, :, :p * PAGE]
        x = x.view(n, hkv, p, PAGE, -1).transpose(1, 2)                                    # [n, p, heads, 16, d]
        x = x[used]
        scale = _pow2(_exponent(x.abs().amax((2, 3))))
        cells.view(torch.uint8)[to[used]] = _rounded(x, scale).view(torch.uint8)
        scales[to[used]] = scale
        back = _read(cells, scales, state["to"]).transpose(1, 2)
        back = torch.nn.functional.pad(back, (0, 0, 0, 0, 0, max(0, keep - back.shape[1])))[:, :keep]
        result.append(torch.where(slot[0, :, :, None, None] < lens[:, None, None, None], back, torch.zeros((), device=back.device)).to(torch.bfloat16))
    return tuple(result)


# ----------------------------------------------------------------------------- in 64 bits
def _nearest8(x):
    """The e4m3 number next to each of ``x`` (fp64), ties to the even one."""
    m, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _block_scale(a):
    e = torch.ceil(torch.log2(a.clamp(min=1e-300) / 448.0))
    e = torch.where(torch.ldexp(torch.full_like(e, 448.0), e.int() - 1) >= a, e - 1, e)        # logarithms next to a power of two
    e = torch.where(torch.ldexp(torch.full_like(e, 448.0), e.int()) < a, e + 1, e)
    return torch.ldexp(torch.ones_like(e), e.clamp(LOW, HIGH).int())


def exact(case, seed):
    state = prepare(case, seed)
    lens, rows, hkv, g, d = state["lens"], state["rows"], case["hkv"], case["g"], case["d"]
    dev = state["k_raw"].device
    tables = state["tables"].cpu().tolist()

    def tokens(i, n, h, which):
        """Values of the first ``n`` tokens of sequence ``i`` and head ``h``."""
        at = torch.tensor(tables[i][:(n + PAGE - 1) // PAGE], device=dev)
        raw = state[which + "_raw"].view(torch.uint8)[:, h][at].view(torch.float8_e4m3fn).double()
        if which == "v":
            raw = raw.transpose(1, 2)
        return (raw * state[which + "s"][:, h][at].double()[:, None, None]).reshape(-1, d)[:n]

    if case["op"] == "write":
        half = case["rot"] // 2
        cos, sin = state["rope"].double()[state["positions"].long()][:, None].split(half, -1)

        def turned(x, w):
            x = x.double()
            if w is not None:
                x = x / ((x ** 2).sum(-1, keepdim=True) / d + 1e-6).sqrt() * w.double()
            y = x.clone()
            y[..., :half] = x[..., :half] * cos - x[..., half:2 * half] * sin
            y[..., half:2 * half] = x[..., half:2 * half] * cos + x[..., :half] * sin
            return y
        results = [turned(state["q"], state["norms"][0])]
        n = state["touched"].shape[0]
        off = state["slots"].long() % PAGE
        for x, which in ((turned(state["key"], state["norms"][1]), "k"), (state["value"].double(), "v")):
            raw = state[which + "_raw"].view(torch.uint8)[state["touched"][:, 0].long()].view(torch.float8_e4m3fn).double()
            raw = raw if which == "k" else raw.transpose(2, 3)
            old = state[which + "s"][state["touched"][:, 0].long()].double()
            fresh = torch.zeros(n, PAGE, hkv, d, dtype=torch.float64, device=dev)
            fresh[state["page_of_row"], off] = x
            begun = state["held"] > 0
            scale = _block_scale(fresh.abs().amax((1, 3)))
            scale = torch.where(begun[:, None] & (old > scale), old, scale)
            value = _nearest8(fresh / scale[:, None, :, None])
            keep = torch.arange(PAGE, device=dev)[None] < state["held"][:, None]
            moved = _nearest8(raw.transpose(1, 2) * (old / scale)[:, None, :, None])
            value = torch.where(keep[:, :, None, None], moved, value) * scale[:, None, :, None]
            value[torch.arange(PAGE, device=dev)[None] >= state["holds"][:, None]] = 0.0
            results.append(value)
        return tuple(results)
    if case["op"] == "evict":
        import numpy as np
        n, keep = len(lens), case["keep"]
        kept = np.full((n, hkv, keep), -1, np.int32)
        out_w = torch.zeros(n, hkv, keep, dtype=torch.float64)
        both = [torch.zeros(n, keep, hkv, d, dtype=torch.float64) for _ in range(2)]
        w = state["weights"].cpu().numpy().astype(np.float64)
        for i, m in enumerate(lens):
            for h in range(hkv):
                if m <= keep:
                    pos = np.arange(m)
                else:
                    mid = np.arange(case["sink"], m - case["recent"])
                    best = mid[np.lexsort((mid, -w[i, h, mid]))][:keep - case["sink"] - case["recent"]]
                    pos = np.sort(np.concatenate([np.arange(case["sink"]), best, np.arange(m - case["recent"], m)]))
                kept[i, h, :len(pos)] = pos
                out_w[i, h, :len(pos)] = torch.from_numpy(w[i, h, pos])
                for which, to in zip("kv", both):
                    x = tokens(i, m, h, which)[torch.from_numpy(pos).to(dev)]
                    full = torch.nn.functional.pad(x, (0, 0, 0, -len(pos) % PAGE)).view(-1, PAGE, d)
                    s = _block_scale(full.abs().amax((1, 2)))[:, None, None]
                    to[i, :len(pos), h] = ((_nearest8(full / s) * s).view(-1, d)[:len(pos)]).cpu()
        return (torch.tensor([min(m, keep) for m in lens], dtype=torch.int32), torch.from_numpy(kept), out_w, both[0], both[1])
    q = state["q"].double()
    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    weights = state["weights"].double() if case["op"] == "weigh" else None
    first = 0
    for i, (n, r) in enumerate(zip(lens, rows)):
        for h in range(hkv):
            k, v = tokens(i, n, h, "k"), tokens(i, n, h, "v")
            for lo in range(0, r, 2048):
                m = min(2048, r - lo)
                seen = torch.arange(n, device=dev)[None] - (n - r + lo + torch.arange(m, device=dev))[:, None]
                gone = (seen > 0) | (seen <= -case["window"] if case["window"] else torch.zeros_like(seen, dtype=torch.bool))
                for e in range(g):
                    s = q[first + lo:first + lo + m, h * g + e] @ k.t() / math.sqrt(d)
                    p = torch.softmax(s.masked_fill(gone, float("-inf")), 1)
                    out[first + lo:first + lo + m, h * g + e] = p @ v
                    if weights is not None:
                        weights[i, h, :n] += p.sum(0)
        first += r
    return out if weights is None else (out, weights)

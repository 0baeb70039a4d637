"""The block-scaled FP8 cache on the GPU against 64-bit forms: writing, reading, attention, weights, eviction, and a run of them together."""
import pytest
import torch

from atlas_b200 import ops
from atlas_b200.models.batch import ForwardBatch
from kv_scaled_cases import (BS, FP8, attention64, attention_bound, dequant, evict64, make_cache, nearest_e4m3, power_scale, tables_for)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def batch_of(lens, rows, tables, device=DEV):
    nd = 0
    while nd < len(rows) and rows[nd] == 1:
        nd += 1
    T = sum(rows)
    pos = torch.cat([torch.arange(n - r, n) for n, r in zip(lens, rows)] + [torch.zeros(0, dtype=torch.long)]).to(torch.int32)
    return ForwardBatch(input_ids=torch.zeros(T, dtype=torch.int64, device=device), positions=pos.to(device),
                        slot_mapping=torch.full((T,), -1, dtype=torch.int32, device=device), block_tables=tables,
                        seq_lens=torch.tensor(lens, dtype=torch.int32, device=device),
                        query_start_loc=torch.tensor([0] + torch.tensor(rows).cumsum(0).tolist(), dtype=torch.int32, device=device),
                        num_decodes=nd, max_query_len=max(rows), max_seq_len=max(lens), seq_lens_host=list(lens), query_lens_host=list(rows))


def slots_of(tables, lens, rows):
    out = []
    for i, (n, r) in enumerate(zip(lens, rows)):
        for p in range(n - r, n):
            out.append(int(tables[i, p // BS]) * BS + p % BS)
    return torch.tensor(out, dtype=torch.int32)


# ----------------------------------------------------------------------------- writing
@pytest.mark.parametrize("d,hkv,g,rot,norm,plus_one,lens,rows", [
    (128, 8, 4, 128, False, False, [16, 33, 1, 200], [1, 1, 1, 1]),
    (128, 2, 1, 64, True, False, [40, 5, 17], [40, 5, 1]),
    (64, 1, 16, 16, True, True, [1, 100], [1, 37]),
    (256, 2, 8, 64, True, True, [530, 29], [517, 2]),
    (64, 5, 3, 0, False, False, [48, 31], [3, 15]),
    (256, 1, 1, 256, False, False, [16], [16]),
    (128, 3, 5, 128, True, False, [700, 64], [600, 1]),
])
def test_write_sets_and_raises_block_scales(d, hkv, g, rot, norm, plus_one, lens, rows):
    gen = torch.Generator().manual_seed(d + hkv)
    tables, nb = tables_for(lens, gen, DEV)
    k, v, ks, vs = make_cache(nb, hkv, d, gen, DEV)
    before = {n: (dequant(c, s, torch.arange(nb), nb * BS), s.clone(), c.view(torch.uint8).cpu().clone()) for n, c, s in (("k", k, ks), ("v", v, vs))}
    T = sum(rows)
    qkv = torch.randn(T, (g + 2) * hkv * d, generator=gen)
    qkv *= torch.exp2(torch.randint(-12, 6, (T, 1), generator=gen).float())            # rows of very different size in one block
    qkv = qkv.to(torch.bfloat16).to(DEV)
    q, kk, vv = (x.view(T, -1, d) for x in qkv.split([g * hkv * d, hkv * d, hkv * d], 1))
    pos = torch.cat([torch.arange(n - r, n) for n, r in zip(lens, rows)]).to(torch.int32).to(DEV)
    turn = torch.outer(torch.arange(max(lens)).double(), 1e4 ** (-torch.arange(0, max(rot, 2), 2).double() / max(rot, 2)))
    rope = torch.cat([turn.cos(), turn.sin()], 1).float().to(DEV)
    wq, wk = ((torch.randn(d, generator=gen) * 0.3 + (0.0 if plus_one else 1.0)).to(torch.bfloat16).to(DEV) for _ in range(2)) if norm else (None, None)
    slots = slots_of(tables, lens, rows).to(DEV)
    keep = qkv.clone()
    out = ops.qk_norm_rope_kv_write(q, kk, vv, pos, rope, rot, k, v, slots, ks, vs, wq, wk, 1e-6, plus_one)
    torch.cuda.synchronize()
    assert torch.equal(qkv, keep)

    def turned(x, w):
        x = x.double().cpu()
        if w is not None:
            w = w.double().cpu() + (1.0 if plus_one else 0.0)
            x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
        if not rot:
            return x
        cs = rope.cpu().double()[pos.cpu().long()][:, None]
        c, s, a, b = cs[..., :rot // 2], cs[..., rot // 2:], x[..., :rot // 2], x[..., rot // 2:rot]
        return torch.cat([a * c - b * s, b * c + a * s, x[..., rot:]], -1)

    want = turned(q, wq)
    size = want.abs().amax(-1, keepdim=True)
    assert (out.double().cpu() - want).abs().le(2.0 ** -8 * want.abs() + 2.0 ** -20 * size).all()
    slots = slots.cpu().tolist()
    for name, x, cache, scales in (("k", turned(kk, wk), k, ks), ("v", vv.double().cpu(), v, vs)):
        now = dequant(cache, scales, torch.arange(nb), nb * BS)
        old, old_scale, old_codes = before[name]
        fuzzy = name == "k" and (norm or rot)                    # fp32 operations before the rounding
        written = {}
        for t, s in enumerate(slots):
            written.setdefault(s // BS, []).append((s % BS, t))
        for blk, cells in written.items():
            first = cells[0][0]
            rows_ = torch.stack([x[t] for _, t in cells])         # [n, hkv, d]
            scale = power_scale(rows_.abs().amax((0, 2)))
            if first:
                scale = torch.maximum(scale, old_scale[blk].cpu().double())
            got = scales[blk].cpu().double()
            if fuzzy:
                near = power_scale(rows_.abs().amax((0, 2)) * (1 + 2.0 ** -18))
                lower = power_scale(rows_.abs().amax((0, 2)) * (1 - 2.0 ** -18))
                if first:
                    near, lower = torch.maximum(near, old_scale[blk].cpu().double()), torch.maximum(lower, old_scale[blk].cpu().double())
                assert ((got == near) | (got == lower)).all()
            else:
                assert torch.equal(got, scale)
            s = got[None, :, None]
            for off, t in cells:
                val = now[blk * BS + off][None]
                if fuzzy:
                    err = (val - x[t][None]).abs()
                    assert err.le((2.0 ** -4 + 2.0 ** -18) * x[t][None].abs() + 2.0 ** -10 * s + 2.0 ** -20 * x[t].abs().amax(-1)[None, :, None]).all()
                else:
                    assert torch.equal(val, nearest_e4m3(x[t][None] / s) * s)
            for off in range(first):                               # what the block held moved to the new scale
                was = old[blk * BS + off][None]
                assert torch.equal(now[blk * BS + off][None], nearest_e4m3(was / s) * s)
            last = cells[-1][0]
            assert torch.equal(cache.view(torch.uint8).cpu()[blk, last + 1:], old_codes[blk, last + 1:])
        for blk in set(range(nb)) - set(written):
            assert torch.equal(cache.view(torch.uint8).cpu()[blk], old_codes[blk]) and torch.equal(scales[blk].cpu(), old_scale[blk].cpu())


def test_write_skips_padding_rows_and_blocks_outside_of_the_pool():
    gen = torch.Generator().manual_seed(3)
    k, v, ks, vs = make_cache(4, 2, 128, gen, DEV)
    old = k.view(torch.uint8).clone(), v.view(torch.uint8).clone(), ks.clone(), vs.clone()
    x = torch.randn(3, 2, 128, generator=gen).to(torch.bfloat16).to(DEV)
    slots = torch.tensor([-1, -5, 64], dtype=torch.int32, device=DEV)
    ops.qk_norm_rope_kv_write(x, x, x, None, None, 0, k, v, slots, ks, vs)
    torch.cuda.synchronize()
    for a, b in zip((k.view(torch.uint8), v.view(torch.uint8), ks, vs), old):
        assert torch.equal(a, b)


@pytest.mark.parametrize("value,scale", [(0.0, 2.0 ** -60), (448.0, 1.0), (450.0, 2.0), (1e-30, 2.0 ** -60), (3e38, 2.0 ** 60), (float("inf"), 2.0 ** 60)])
def test_scales_at_their_ends(value, scale):
    k, v, ks, vs = make_cache(1, 1, 64, torch.Generator().manual_seed(0), DEV)
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device=DEV)
    x[0, 0, 5] = value
    ops.qk_norm_rope_kv_write(x, x, x, None, None, 0, k, v, torch.zeros(1, dtype=torch.int32, device=DEV), ks, vs)
    exact = float(x[0, 0, 5])
    want = float(power_scale(torch.tensor(exact)))
    assert float(ks[0, 0]) == float(vs[0, 0]) == want
    assert value in (450.0,) or want == scale


# ----------------------------------------------------------------------------- reading
@pytest.mark.parametrize("d,hkv,lens,max_len", [(64, 3, [1, 0, 40, 17], 40), (128, 8, [33, 100], 50), (256, 1, [16, 15], 37)])
def test_read_gives_the_cache_exactly(d, hkv, lens, max_len):
    gen = torch.Generator().manual_seed(1)
    tables, nb = tables_for(lens, gen, DEV)
    k, v, ks, vs = make_cache(nb, hkv, d, gen, DEV, spread=20)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    got = ops.kv_read(k, v, tables, n, max_len, ks, vs)
    for x, c, s in zip(got, (k, v), (ks, vs)):
        assert x.shape == (len(lens), max_len, hkv, d) and x.dtype == torch.bfloat16
        for i, m in enumerate(lens):
            m = min(m, max_len)
            assert torch.equal(x[i, :m].double().cpu(), dequant(c, s, tables[i], m)) and not x[i, m:].any()


# ----------------------------------------------------------------------------- attention
ATTEND = [
    # decode only
    (128, 8, 4, [77], [1], 0),
    (128, 8, 4, [1, 16, 17, 300, 2], [1] * 5, 0),
    (128, 1, 1, [5000], [1], 0),
    (64, 2, 7, [33, 1000, 15], [1] * 3, 0),
    (256, 2, 8, [129, 65, 700], [1] * 3, 0),
    (128, 2, 16, [40, 513], [1] * 2, 0),
    (256, 1, 16, [100, 31], [1] * 2, 0),
    (64, 1, 40, [70, 16], [1] * 2, 0),
    (128, 4, 5, [400, 16, 50], [1] * 3, 33),
    (64, 3, 2, [257] * 40, [1] * 40, 1),
    (64, 1, 2, [1 + (7 * i) % 50 for i in range(300)], [1] * 300, 0),
    (64, 1, 4, [30000, 20], [1] * 2, 0),
    # chunks
    (128, 8, 4, [300, 129], [300, 129], 0),
    (128, 2, 8, [40, 700], [2, 100], 0),
    (64, 4, 3, [513], [513], 0),
    (256, 2, 8, [530], [517], 0),
    (256, 1, 1, [200, 2], [200, 2], 0),
    (128, 1, 5, [260, 33], [250, 33], 0),
    (128, 2, 16, [130], [65], 0),
    (128, 1, 128, [20], [9], 0),
    (128, 4, 4, [600, 250], [600, 100], 100),
    (64, 2, 1, [400], [300], 17),
    # few rows behind many keys: shares of the keys
    (128, 1, 4, [5000, 700], [40, 2], 0),
    (64, 2, 8, [3000], [3], 0),
    (256, 1, 8, [4000, 130, 2000], [1, 5, 40], 0),
    (128, 2, 4, [9000], [300], 2500),
    # both
    (128, 4, 7, [90, 2000, 300, 65], [1, 1, 300, 3], 0),
    (256, 2, 2, [70, 200], [1, 130], 50),
    (64, 8, 8, [1, 17, 100], [1, 1, 2], 0),
]


@pytest.mark.parametrize("weigh", [False, True])
@pytest.mark.parametrize("d,hkv,g,lens,rows,window", ATTEND)
def test_attention_and_weights(d, hkv, g, lens, rows, window, weigh):
    check_attention(d, hkv, g, lens, rows, window, weigh)


def check_attention(d, hkv, g, lens, rows, window, weigh, smallest=False):
    gen = torch.Generator().manual_seed(d * hkv + g)
    tables, nb = tables_for(lens, gen, DEV, extra_cols=2)
    k, v, ks, vs = make_cache(nb, hkv, d, gen, DEV)
    # what stands behind a sequence's end is not a number
    for i, n in enumerate(lens):
        if n % BS:
            blk = int(tables[i, n // BS])
            k.view(torch.uint8)[blk, n % BS:] = 0x7F
            v.view(torch.uint8)[blk, n % BS:] = 0xFF
    T = sum(rows)
    q = (torch.randn(T, hkv * g, d, generator=gen) * torch.exp2(torch.randint(-6, 2, (T, hkv * g, 1), generator=gen).float())).to(torch.bfloat16).to(DEV)
    batch = batch_of(lens, rows, tables)
    scale = d ** -0.5
    weights = start = None
    if weigh:
        start = torch.rand(len(lens), hkv, max(lens) + 5, generator=gen)
        weights = start.clone().to(DEV)
    got = ops.paged_attention(q, k, v, batch, scale, ks, vs, window or None, weights=weights)
    torch.cuda.synchronize()
    from atlas_b200.ops import cuda as K
    assert K.check_status() == 0
    out, mag, amp, w = attention64(q, k, v, ks, vs, tables, lens, rows, scale, window)
    bound = attention_bound(out, mag, amp, d)
    if smallest:
        # f16 has steps of 2^-24 below 2^-14: a weight p_j = 2^(s_j + ev_j - M) is off by 2^-25 at most however small it is, so the output by
        # 2^-25 sum_j |code_j| / l over the window's tokens.  The token that the reference M comes from has p >= 1, l >= 2^-ev of it, and
        # 448 * 2^ev < 2 max |v| there (a block's largest code is above 224): n 2^-24 max |v| altogether.
        bound = bound + window * 2.0 ** -24 * float((v.float().abs().nan_to_num(0.0).amax((1, 3)) * vs).max())
    assert (got.double().cpu() - out).abs().le(bound).all()
    if weigh:
        r0 = 0
        for i, (n, r) in enumerate(zip(lens, rows)):
            have = weights[i].double().cpu()
            want = start[i].double()
            want[:, :n] += w[i]
            rel = 4 * (d / 16 + 8) * 2.0 ** -23 * (float(amp[r0:r0 + r].max()) + 2.0) + 2.0 ** -20
            # each weight by the scores' and the sums' errors, the sum over rows and heads and the running sum in fp32
            assert (have[:, :n] - want[:, :n]).abs().le(rel * w[i] + (r * g / 32 + 8) * 2.0 ** -23 * want[:, :n] + 1e-37).all()
            assert torch.equal(have[:, n:], want[:, n:])
            r0 += r


@pytest.mark.parametrize("weigh", [False, True])
@pytest.mark.parametrize("d,hkv,g,lens,rows,window", [
    # one long sequence among many short ones: hundreds of pieces for one pair, one for the others, joined by threads and by blocks
    (64, 1, 2, [16] * 600 + [6000], [1] * 601, 0),
    (64, 1, 2, [16] * 40 + [20000], [1] * 41, 0),
    (128, 2, 6, [3000, 17, 900] * 4, [1] * 12, 0),
    (256, 1, 9, [2500, 1, 40], [1] * 3, 0),
    # several items a CTA, tiles without rows or keys among them
    (64, 8, 8, [200] * 12, [200] * 12, 0),
    (128, 8, 3, [90, 400, 43, 129] * 8, [43, 129, 43, 129] * 8, 0),
    (128, 16, 4, [300, 5, 64] * 6, [256, 5, 1] * 6, 40),
    (256, 8, 3, [90, 300, 43] * 8, [43, 129, 43] * 8, 0),
])
def test_attention_of_many_pieces_and_items(d, hkv, g, lens, rows, window, weigh):
    check_attention(d, hkv, g, lens, rows, window, weigh, smallest=window > 0)


def test_scales_far_apart_keep_small_values():
    """One page's values are 2^-40 of the others', and its token has all the weight."""
    gen = torch.Generator().manual_seed(5)
    for rows in ([1], [20]):
        tables, nb = tables_for([100], gen, DEV)
        k, v, ks, vs = make_cache(nb, 2, 128, gen, DEV)
        vs[int(tables[0, 2])] *= 2.0 ** -40
        q = torch.zeros(sum(rows), 4, 128)
        key = dequant(k, ks, tables[0], 100)[37]                      # [2, 128]
        q[:] = (key / key.norm(dim=-1, keepdim=True)).repeat_interleave(2, 0).float() * 400.0
        q = q.to(torch.bfloat16).to(DEV)
        got = ops.paged_attention(q, k, v, batch_of([100], rows, tables), 1.0, ks, vs)
        out, mag, amp, _ = attention64(q, k, v, ks, vs, tables, [100], rows, 1.0)
        assert out.abs().max() < 1e-8
        assert (got.double().cpu() - out).abs().le(attention_bound(out, mag, amp, 128)).all()


def test_empty_decode_sequences_give_zeros():
    gen = torch.Generator().manual_seed(6)
    tables, nb = tables_for([30, 0, 5], gen, DEV)
    k, v, ks, vs = make_cache(nb, 2, 64, gen, DEV)
    q = torch.randn(3, 4, 64, generator=gen).to(torch.bfloat16).to(DEV)
    batch = batch_of([30, 1, 5], [1, 1, 1], tables)
    batch.seq_lens = torch.tensor([30, 0, 5], dtype=torch.int32, device=DEV)
    w = torch.ones(3, 2, 30, device=DEV)
    got = ops.paged_attention(q, k, v, batch, 0.1, ks, vs, weights=w)
    assert not got[1].any() and got[0].any() and got[2].any()
    assert torch.equal(w[1], torch.ones(2, 30, device=DEV))


# ----------------------------------------------------------------------------- eviction
@pytest.mark.parametrize("d,hkv,lens,keep,sink,recent", [
    (128, 2, [100, 37, 64], 37, 4, 8), (64, 1, [1000, 3], 16, 0, 0), (256, 3, [333], 100, 0, 100), (128, 1, [5000, 40, 1], 1000, 16, 1),
    (64, 2, [50], 1, 1, 0), (128, 2, [70], 70, 3, 3), (64, 1, [20000], 333, 1, 30), (64, 1, [9000, 100], 700, 3, 9), (64, 20, [5000], 40, 0, 4)])
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
def test_evict_keeps_the_heaviest_in_order(d, hkv, lens, keep, sink, recent, kind):
    gen = torch.Generator().manual_seed(keep)
    B = len(lens)
    tables, nb = tables_for(lens, gen, DEV)
    to, spare = tables_for([min(n, keep) for n in lens], gen, DEV)
    k, v, ks, vs = make_cache(nb + spare, hkv, d, gen, DEV)
    to = to + nb
    w = torch.rand(B, hkv, max(lens) + 3, generator=gen)
    if kind == "ties":
        w = (w * 4).floor() / 4
    elif kind == "odd":
        w = torch.where(w < 0.2, torch.full_like(w, float("nan")), torch.where(w < 0.4, torch.full_like(w, float("inf")), w - 0.7))
        w[..., ::7] = -0.0
        w[..., 1::7] = 0.0
    old = k.view(torch.uint8).clone(), v.view(torch.uint8).clone(), ks.clone(), vs.clone()
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    new_lens, kept, out_w = ops.kv_evict(k, v, ks, vs, tables, n, w.to(DEV), keep, to, sink=sink, recent=recent)
    torch.cuda.synchronize()
    assert new_lens.tolist() == [min(x, keep) for x in lens]
    for a, b in zip((k.view(torch.uint8), v.view(torch.uint8), ks, vs), old):
        assert torch.equal(a[:nb], b[:nb])
    for i, m in enumerate(lens):
        s = min(m, keep)
        for h in range(hkv):
            pos = evict64(w[i, h], m, keep, sink, recent)
            assert kept[i, h, :s].tolist() == pos and (kept[i, h, s:] == -1).all()
            assert torch.equal(out_w[i, h, :s].cpu().view(torch.int32), w[i, h, pos].view(torch.int32)) and not out_w[i, h, s:].any()
            for c, sc, oc, osc in ((k, ks, old[0], old[2]), (v, vs, old[1], old[3])):
                was = dequant(oc.view(FP8), osc, tables[i], m)[pos][:, h]
                pages = torch.nn.functional.pad(was, (0, 0, 0, -s % BS)).view(-1, BS, d)
                scale = power_scale(pages.abs().amax((1, 2)))[:, None, None]
                want = (nearest_e4m3(pages / scale) * scale).view(-1, d)[:s]
                assert torch.equal(dequant(c, sc, to[i], s)[:, h], want)


# ----------------------------------------------------------------------------- together, captured, on other streams
def _steps(lens0, hkv, g, d, steps, seed):
    """Prompts, decode steps with weights, an eviction, more decode steps: the outputs of every stage."""
    gen = torch.Generator().manual_seed(seed)
    B = len(lens0)
    cap = [n + 2 * steps for n in lens0]
    tables, nb = tables_for(cap, gen, DEV)
    keep = 32
    to, spare = tables_for([keep + steps] * B, gen, DEV)
    to = to + nb
    k, v, ks, vs = make_cache(nb + spare, hkv, d, gen, DEV)
    turn = torch.outer(torch.arange(max(cap)).double(), 1e4 ** (-torch.arange(0, d, 2).double() / d))
    rope = torch.cat([turn.cos(), turn.sin()], 1).float().to(DEV)
    weights = torch.zeros(B, hkv, max(cap), device=DEV)
    outs = []

    def step(lens, rows, tabs, positions, w):
        T = sum(rows)
        qkv = torch.randn(T, (g + 2) * hkv * d, generator=gen).to(torch.bfloat16).to(DEV)
        q, kk, vv = (x.view(T, -1, d) for x in qkv.split([g * hkv * d, hkv * d, hkv * d], 1))
        q = ops.qk_norm_rope_kv_write(q, kk, vv, positions, rope, d, k, v, slots_of(tabs, lens, rows).to(DEV), ks, vs)
        o = ops.paged_attention(q, k, v, batch_of(lens, rows, tabs), d ** -0.5, ks, vs, weights=w)
        ref = attention64(q, k, v, ks, vs, tabs, lens, rows, d ** -0.5)
        assert (o.double().cpu() - ref[0]).abs().le(attention_bound(*ref[:3], d)).all()
        outs.append(o)
    lens = list(lens0)
    step(lens, lens, tables, torch.cat([torch.arange(n) for n in lens]).to(torch.int32).to(DEV), weights)
    for _ in range(steps):
        lens = [n + 1 for n in lens]
        step(lens, [1] * B, tables, torch.tensor([n - 1 for n in lens], dtype=torch.int32, device=DEV), weights)
    total = weights.sum().item()
    rows_seen = sum(lens0) + B * steps
    assert abs(total - rows_seen * hkv * g) < 1e-4 * rows_seen * hkv * g            # every row's weights sum to one
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    new_lens, kept, w2 = ops.kv_evict(k, v, ks, vs, tables, n, weights, keep, to, sink=2, recent=4)
    short = new_lens.tolist()
    w3 = torch.cat([w2, torch.zeros(B, hkv, steps, device=DEV)], 2).contiguous()
    for i in range(steps):                                                           # positions go on, the cache is shorter
        lens, short = [x + 1 for x in lens], [x + 1 for x in short]
        step(short, [1] * B, to, torch.tensor([x - 1 for x in lens], dtype=torch.int32, device=DEV), w3)
    return outs + [kept, w3]


def test_prompt_decode_evict_decode():
    _steps([70, 45, 20], 2, 4, 128, 5, 0)


def test_repeats_bit_for_bit():
    a, b = _steps([70, 45], 2, 4, 64, 2, 1), _steps([70, 45], 2, 4, 64, 2, 1)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_calls_follow_their_inputs():
    """One decode step (write, attention with weights) and an eviction in a graph, replayed with other inputs on another stream, beside a
    second graph of other sizes."""
    gen = torch.Generator().manual_seed(9)

    def capture(lens, hkv, g, d):
        B = len(lens)
        tables, nb = tables_for([n + 8 for n in lens], gen, DEV)
        to, spare = tables_for([16] * B, gen, DEV)
        to = to + nb
        k, v, ks, vs = make_cache(nb + spare, hkv, d, gen, DEV)
        batch = batch_of(lens, [1] * B, tables)
        batch.max_seq_len = max(lens) + 8
        qkv = torch.randn(B, (g + 2) * hkv, d, generator=gen).to(torch.bfloat16).to(DEV)
        slots = slots_of(tables, lens, [1] * B).to(DEV)
        w = torch.zeros(B, hkv, max(lens) + 8, device=DEV)

        def call():
            q = ops.qk_norm_rope_kv_write(qkv[:, :g * hkv], qkv[:, g * hkv:(g + 1) * hkv], qkv[:, (g + 1) * hkv:], None, None, 0, k, v, slots, ks, vs)
            o = ops.paged_attention(q, k, v, batch, 0.1, ks, vs, weights=w)
            return (o,) + ops.kv_evict(k, v, ks, vs, tables, batch.seq_lens, w, 16, to, recent=1)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            call()
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = call()
        return gr, outs, call, batch, qkv, slots, w, tables, lens, B
    graphs = [capture([40, 200], 2, 4, 128), capture([90], 1, 8, 64)]
    for step in range(3):
        for gr, outs, call, batch, qkv, slots, w, tables, lens, B in graphs:
            now = [n + step for n in lens]
            batch.seq_lens.copy_(torch.tensor(now, dtype=torch.int32))
            slots.copy_(slots_of(tables, now, [1] * B))
            qkv.copy_(torch.randn(qkv.shape, generator=gen).to(torch.bfloat16))
            w.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for (gr, *_), s in zip(graphs, streams):
        with torch.cuda.stream(s):
            gr.replay()
    torch.cuda.synchronize()
    for gr, outs, call, batch, qkv, slots, w, *_ in graphs:
        got = [x.clone() for x in outs]
        w.zero_()
        want = call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_calls_on_two_streams_do_not_meet():
    gen = torch.Generator().manual_seed(11)
    cases = []
    for lens, rows in (([3000], [1]), ([500, 900], [1, 1]), ([300], [300])):
        tables, nb = tables_for(lens, gen, DEV)
        c = make_cache(nb, 4, 128, gen, DEV)
        q = torch.randn(sum(rows), 16, 128, generator=gen).to(torch.bfloat16).to(DEV)
        b = batch_of(lens, rows, tables)
        cases.append((q, c, b, ops.paged_attention(q, c[0], c[1], b, 0.09, c[2], c[3])))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for s, (q, c, b, _) in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(ops.paged_attention(q, c[0], c[1], b, 0.09, c[2], c[3]))
        torch.cuda.synchronize()
        assert all(torch.equal(x, case[3]) for x, case in zip(got, cases))

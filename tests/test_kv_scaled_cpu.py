"""The block-scaled FP8 cache without a GPU: the plain forms against 64-bit ones, what the calls refuse, and the checked mode."""
import pytest
import torch

from atlas_b200 import ops
from atlas_b200.models.batch import ForwardBatch
from atlas_b200.ops import checked, cuda as K, cuda_scaled as CS
from kv_scaled_cases import BS, attention64, attention_bound, dequant, evict64, make_cache, nearest_e4m3, power_scale, tables_for


def batch_of(lens, rows, tables):
    nd = 0
    while nd < len(rows) and rows[nd] == 1:
        nd += 1
    return ForwardBatch(input_ids=torch.zeros(sum(rows), dtype=torch.int64), positions=None, slot_mapping=None, block_tables=tables,
                        seq_lens=torch.tensor(lens, dtype=torch.int32),
                        query_start_loc=torch.tensor([0] + torch.tensor(rows).cumsum(0).tolist(), dtype=torch.int32), num_decodes=nd,
                        max_query_len=max(rows), max_seq_len=max(lens), seq_lens_host=list(lens), query_lens_host=list(rows))


def test_scale_is_the_smallest_power_that_holds_the_block():
    a = torch.tensor([0.0, 1.0, 448.0, 448.00003, 449.0, 224.0, 1e-38, 2.0 ** -60 * 448, 3e38, float("inf")])
    from atlas_b200.ops.reference_scaled import block_scale
    assert torch.equal(block_scale(a).double(), power_scale(a))
    assert block_scale(torch.tensor(448.0)) == 1.0 and block_scale(torch.tensor(448.00003)) == 2.0


@pytest.mark.parametrize("lens,rows", [([16, 33, 5], [16, 20, 1]), ([1, 40], [1, 7])])
def test_write_and_read(lens, rows):
    gen = torch.Generator().manual_seed(0)
    tables, nb = tables_for(lens, gen, "cpu")
    k, v, ks, vs = make_cache(nb, 2, 64, gen, "cpu", kernel_layout=False)
    old = [dequant(c, s, torch.arange(nb), nb * BS) for c, s in ((k, ks), (v, vs))]
    old_scale = ks.clone(), vs.clone()
    T = sum(rows)
    x = (torch.randn(T, 2, 64, generator=gen) * torch.exp2(torch.randint(-9, 4, (T, 1, 1), generator=gen).float())).to(torch.bfloat16)
    slots = torch.tensor([int(tables[i, p // BS]) * BS + p % BS for i, (n, r) in enumerate(zip(lens, rows)) for p in range(n - r, n)], dtype=torch.int32)
    out = ops.qk_norm_rope_kv_write(x, x, -x, None, None, 0, k, v, slots, ks, vs)
    assert torch.equal(out, x)
    for sign, c, s, was, was_s in ((1, k, ks, old[0], old_scale[0]), (-1, v, vs, old[1], old_scale[1])):
        now = dequant(c, s, torch.arange(nb), nb * BS)
        by_block = {}
        for t, slot in enumerate(slots.tolist()):
            by_block.setdefault(slot // BS, []).append((slot % BS, t))
        for blk, cells in by_block.items():
            rows_ = torch.stack([x[t].double() for _, t in cells])
            want = power_scale(rows_.abs().amax((0, 2)))
            if cells[0][0]:
                want = torch.maximum(want, was_s[blk].double())
            assert torch.equal(s[blk].double(), want)
            for off, t in cells:
                assert torch.equal(now[blk * BS + off], nearest_e4m3(sign * x[t].double() / want[:, None]) * want[:, None])
            for off in range(cells[0][0]):
                assert torch.equal(now[blk * BS + off], nearest_e4m3(was[blk * BS + off] / want[:, None]) * want[:, None])
    n = torch.tensor(lens, dtype=torch.int32)
    kk, vv = ops.kv_read(k, v, tables, n, 20, ks, vs)
    for i, m in enumerate(lens):
        m = min(m, 20)
        assert torch.equal(kk[i, :m].double(), dequant(k, ks, tables[i], m)) and not kk[i, m:].any()
        assert torch.equal(vv[i, :m].double(), dequant(v, vs, tables[i], m)) and not vv[i, m:].any()


@pytest.mark.parametrize("window", [0, 9])
def test_attention_and_weights(window):
    gen = torch.Generator().manual_seed(1)
    lens, rows = [33, 17, 40], [1, 17, 12]
    tables, nb = tables_for(lens, gen, "cpu")
    k, v, ks, vs = make_cache(nb, 2, 64, gen, "cpu", kernel_layout=False)
    q = torch.randn(sum(rows), 6, 64, generator=gen).to(torch.bfloat16)
    w = torch.ones(3, 2, 41)
    got = ops.paged_attention(q, k, v, batch_of(lens, rows, tables), 0.125, ks, vs, window or None, weights=w)
    out, mag, amp, sums = attention64(q, k, v, ks, vs, tables, lens, rows, 0.125, window)
    assert (got.double() - out).abs().le(attention_bound(out, mag, amp, 64)).all()
    for i, n in enumerate(lens):
        # p is off by its score's rounding: (64 + 8) fp32 steps of the scores' magnitude, twice, as an exponent
        tol = 4 * 72 * 2.0 ** -23 * (float(amp.max()) + 2.0)
        assert (w[i, :, :n].double() - 1.0 - sums[i]).abs().le(tol * sums[i] + 2.0 ** -20 * (1 + sums[i])).all() and w[i, :, n:].eq(1).all()


def test_evict_by_weight():
    gen = torch.Generator().manual_seed(2)
    lens, keep = [50, 20, 33], 24
    tables, nb = tables_for(lens, gen, "cpu")
    to, spare = tables_for([keep] * 3, gen, "cpu")
    to = to + nb
    k, v, ks, vs = make_cache(nb + spare, 2, 64, gen, "cpu", kernel_layout=False)
    w = (torch.rand(3, 2, 50, generator=gen) * 6).floor()
    n, kept, out_w = ops.kv_evict(k, v, ks, vs, tables, torch.tensor(lens, dtype=torch.int32), w, keep, to, sink=2, recent=5)
    assert n.tolist() == [24, 20, 24]
    for i, m in enumerate(lens):
        s = min(m, keep)
        for h in range(2):
            pos = evict64(w[i, h], m, keep, 2, 5)
            assert kept[i, h, :s].tolist() == pos and (kept[i, h, s:] == -1).all()
            assert torch.equal(out_w[i, h, :s], w[i, h, pos])
            was = dequant(v, vs, tables[i], m)[pos][:, h]
            now = dequant(v, vs, to[i], s)[:, h]
            page = torch.nn.functional.pad(was, (0, 0, 0, -s % BS)).view(-1, BS, 64)
            scale = power_scale(page.abs().amax((1, 2)))[:, None, None]
            assert torch.equal(now, (nearest_e4m3(page / scale) * scale).view(-1, 64)[:s])


# ----------------------------------------------------------------------------- refusals (before anything is launched)
def parts(d=64, nb=4, hkv=2, bs=16):
    k = torch.zeros(nb, hkv, bs, d, dtype=torch.uint8).view(K.FP8).permute(0, 2, 1, 3)
    v = torch.zeros(nb, hkv, d, bs, dtype=torch.uint8).view(K.FP8).permute(0, 3, 1, 2)
    return (k, v) + CS.alloc_kv_scales(nb, hkv, "cpu")


def write(k_cache, v_cache, ks, vs, T=2, hq=4, d=64, **kw):
    a = dict(q=torch.zeros(T, hq, d, dtype=torch.bfloat16), k=torch.zeros(T, 2, d, dtype=torch.bfloat16), v=torch.zeros(T, 2, d, dtype=torch.bfloat16),
             positions=torch.zeros(T, dtype=torch.int32), rope=torch.zeros(8, 32), rot=32, slots=torch.zeros(T, dtype=torch.int32), norms=(None, None))
    a.update(kw)
    return CS.qk_norm_rope_kv_write(a["q"], a["k"], a["v"], a["positions"], a["rope"], a["rot"], k_cache, v_cache, a["slots"], ks, vs,
                                    *a["norms"])


BF = torch.bfloat16


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(2, 4, 64)), dict(q=torch.zeros(3, 4, 64, dtype=BF)), dict(k=torch.zeros(2, 3, 64, dtype=BF)), dict(v=torch.zeros(2, 2, 32, dtype=BF)),
    dict(k=torch.zeros(2, 2, 128, dtype=BF)[..., ::2]), dict(slots=torch.zeros(2)), dict(slots=torch.zeros(3, dtype=torch.int32)),
    dict(positions=torch.zeros(1, dtype=torch.int32)), dict(rot=66), dict(rot=6), dict(rope=torch.zeros(8, 16)), dict(rope=torch.zeros(8, 32).double()),
    dict(norms=(torch.zeros(64, dtype=BF), None)), dict(norms=(torch.zeros(64), torch.zeros(64)))])
def test_write_refuses(change):
    with pytest.raises(K.KernelError):
        write(*parts(), **change)


def test_caches_refused():
    k, v, ks, vs = parts()
    for bad in ((k, v, ks, 1.0), (k, v, ks.double(), vs), (k, v, ks[:2], vs), (k, v, ks.t(), vs), (v, k, ks, vs), (k.to(torch.bfloat16), v, ks, vs),
                parts(d=96), parts(bs=32), (k.contiguous(), v, ks, vs)):
        with pytest.raises(K.KernelError):
            write(*bad)


def attend(k, v, ks, vs, lens=(20, 5), rows=(1, 1), **kw):
    a = dict(q=torch.zeros(sum(rows), 4, 64, dtype=BF), window=None, weights=None)
    a.update(kw)
    b = batch_of(list(lens), list(rows), a.pop("tables", torch.zeros(len(lens), 2, dtype=torch.int32)))
    return CS.paged_attention(a["q"], k, v, b, 0.1, ks, vs, a["window"], a["weights"])


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(2, 3, 64, dtype=BF)), dict(q=torch.zeros(2, 4, 64)), dict(q=torch.zeros(2, 258, 64, dtype=BF)), dict(window=-1),
    dict(q=torch.zeros(2, 4 * 64 + 4, dtype=BF)[:, :256].view(2, 4, 64)), dict(tables=torch.zeros(1, 2, dtype=torch.int32)),
    dict(tables=torch.zeros(2, 2)), dict(q=torch.zeros(1, 4, 64, dtype=BF)), dict(weights=torch.zeros(2, 2, 19)), dict(weights=torch.zeros(2, 4, 32)),
    dict(weights=torch.zeros(2, 2, 32).double()), dict(weights=torch.zeros(2, 2, 64)[..., ::2])])
def test_attention_refuses(change):
    with pytest.raises(K.KernelError):
        attend(*parts(), **change)


def test_front_end_refuses():
    k, v, ks, vs = parts()
    q = torch.zeros(1, 4, 64, dtype=BF)
    b = batch_of([3], [1], torch.zeros(1, 1, dtype=torch.int32))
    for kw in (dict(chunk=4), dict(sinks=torch.zeros(4)), dict(softcap=1.0), dict(distance=torch.zeros(4, 3))):
        with pytest.raises(ValueError):
            ops.paged_attention(q, k, v, b, 0.1, ks, vs, **kw)
    with pytest.raises(ValueError):
        ops.paged_attention(q, k, v, b, 0.1, 1.0, 1.0, weights=torch.zeros(1, 2, 3))
    with pytest.raises(ValueError):
        ops.qk_norm_rope_kv_write(q, q[:, :2], q[:, :2], None, None, 0, k, v, torch.zeros(1, dtype=torch.int32), ks, vs, rotate=True)
    with pytest.raises(ValueError):
        ops.kv_evict(k, v, ks, vs, b.block_tables, b.seq_lens, torch.zeros(1, 2, 3), 2, b.block_tables, sink=2, recent=1)


def test_evict_and_read_refuse():
    k, v, ks, vs = parts()
    t, n, w = torch.zeros(2, 2, dtype=torch.int32), torch.full((2,), 20, dtype=torch.int32), torch.zeros(2, 2, 32)
    good = dict(tables=t, n=n, w=w, keep=17, to=t, sink=1, recent=1)
    for change in (dict(keep=0), dict(sink=-1), dict(sink=17), dict(to=t[:, :1]), dict(n=n[:1]), dict(n=n.long()), dict(w=w[:1]), dict(w=w.double()),
                   dict(w=torch.zeros(2, 2, 64)[..., ::2]), dict(tables=t.long()), dict(to=t.t()[:, ::1].contiguous().t())):
        a = dict(good, **change)
        with pytest.raises(K.KernelError):
            CS.kv_evict(k, v, ks, vs, a["tables"], a["n"], a["w"], a["keep"], a["to"], a["sink"], a["recent"])
    for a in ((t.long(), n, 4), (t, n[:1], 4), (t, n, -1), (t[0], n, 4)):
        with pytest.raises(K.KernelError):
            CS.kv_read(k, v, *a, ks, vs)
    assert CS.kv_read(k, v, t[:0], n[:0], 4, ks, vs)[0].shape == (0, 4, 2, 64)
    assert write(k, v, ks, vs, T=0).shape == (0, 4, 64)


def test_checked_mode():
    checked.block_runs(torch.tensor([3, 4, 5, -1, 16, 17, -1]), 16)
    for bad in ([3, 4, 40, 5], [3, 5], [4, 3]):
        with pytest.raises(checked.BoundsViolation):
            checked.block_runs(torch.tensor(bad), 16)
    t = torch.tensor([[0, 1], [2, 0]], dtype=torch.int32)
    n = torch.tensor([20, 9], dtype=torch.int32)
    checked.evict(t, n, torch.tensor([[3], [4]], dtype=torch.int32), 5, 16, 16, 32)
    for to in ([[3], [3]], [[1], [4]], [[5], [4]]):
        with pytest.raises(checked.BoundsViolation):
            checked.evict(t, n, torch.tensor(to, dtype=torch.int32), 5, 16, 16, 32)

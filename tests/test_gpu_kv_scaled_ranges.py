"""The block-scaled FP8 cache on the GPU, at the ends of what its calls allow."""
import numpy as np
import pytest
import torch

from atlas_b200 import ops
from atlas_b200.ops import cuda as K
from kv_scaled_cases import BS, FP8, attention64_over, attention_bound, dequant, make_cache, nearest_e4m3, power_scale, tables_for
from test_gpu_kv_scaled import batch_of, check_attention
import test_gpu_kv_scaled as base

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# ----------------------------------------------------------------------------- weights of few rows
@pytest.mark.parametrize("d,hkv,g,lens,rows,window", [
    (128, 8, 4, [4000, 2500], [5, 2], 0),
    (64, 8, 16, [5000], [3], 0),
    (256, 4, 8, [3000, 40, 1500], [2, 3, 16], 0),
    (128, 8, 4, [2000] * 6, [4] * 6, 300),
])
def test_weights_where_one_cta_of_a_pair_has_no_rows(d, hkv, g, lens, rows, window):
    for _ in range(3):
        check_attention(d, hkv, g, lens, rows, window, True, smallest=window > 0)


# ----------------------------------------------------------------------------- table entries outside of the pool
@pytest.mark.parametrize("weigh", [False, True])
@pytest.mark.parametrize("d,hkv,g,lens,rows,window,gone", [
    (128, 2, 4, [100, 40], [1, 1], 0, [(0, 0), (0, 3), (1, 1)]),
    (64, 1, 16, [700, 16], [1, 1], 0, [(0, 0), (0, 20), (0, 43), (1, 0)]),
    (256, 2, 3, [90, 33], [1, 1], 20, [(0, 4), (1, 2)]),
    (128, 2, 4, [300, 40], [300, 17], 0, [(0, 0), (0, 9), (0, 18), (1, 0), (1, 1), (1, 2)]),
    (64, 4, 3, [500], [200], 0, [(0, 3), (0, 4), (0, 25)]),
    (256, 2, 8, [300, 70], [90, 70], 0, [(0, 0), (0, 6), (1, 4)]),
    (256, 1, 4, [400], [300], 50, [(0, 5), (0, 12)]),
    (128, 1, 4, [4000], [30], 0, [(0, i) for i in range(0, 250, 3)]),
    (128, 1, 8, [600, 90], [1, 90], 0, [(0, 30), (1, 0)]),
])
def test_blocks_outside_of_the_pool_are_skipped(d, hkv, g, lens, rows, window, gone, weigh):
    """In every kernel alike: their tokens have no weight, and nothing of what lay in memory before comes in."""
    gen = torch.Generator().manual_seed(d + sum(lens))
    tables, nb = tables_for(lens, gen, DEV, extra_cols=1)
    k, v, ks, vs = make_cache(nb, hkv, d, gen, DEV)
    kk = [dequant(k, ks, t, n) for t, n in zip(tables, lens)]
    vv = [dequant(v, vs, t, n) for t, n in zip(tables, lens)]
    there = [torch.ones(n, dtype=torch.bool) for n in lens]
    for x, (i, page) in enumerate(gone):
        tables[i, page] = (-1, nb, -2 ** 31, 2 ** 31 - 1, -7)[x % 5]
        there[i][page * BS:(page + 1) * BS] = False
    q = torch.randn(sum(rows), hkv * g, d, generator=gen).to(torch.bfloat16).to(DEV)
    start = torch.rand(len(lens), hkv, max(lens) + 3, generator=gen)
    w = start.clone().to(DEV) if weigh else None
    for _ in range(2):
        if weigh:
            w.copy_(start)
        got = ops.paged_attention(q, k, v, batch_of(lens, rows, tables), d ** -0.5, ks, vs, window or None, weights=w)
        r0 = 0
        for i, (n, r) in enumerate(zip(lens, rows)):
            out, mag, amp, sums = attention64_over(q[r0:r0 + r], kk[i], vv[i], d ** -0.5, window, there[i])
            assert (got[r0:r0 + r].double().cpu() - out).abs().le(attention_bound(out, mag, amp, d)).all()
            if weigh:
                have, want = w[i].double().cpu(), start[i].double()
                want[:, :n] += sums
                rel = 4 * (d / 16 + 8) * 2.0 ** -23 * (float(amp.max()) + 2.0) + 2.0 ** -20
                assert (have[:, :n] - want[:, :n]).abs().le(rel * sums + (r * g / 32 + 8) * 2.0 ** -23 * want[:, :n] + 1e-37).all()
                assert torch.equal(have[:, n:], want[:, n:])
            r0 += r
    assert K.check_status() == 0


# ----------------------------------------------------------------------------- values of very different size
def _check(q, k, v, ks, vs, tables, lens, rows, scale, window=0):
    got = ops.paged_attention(q, k, v, batch_of(lens, rows, tables), scale, ks, vs, window or None)
    assert K.check_status() == 0
    r0 = 0
    for i, (n, r) in enumerate(zip(lens, rows)):
        out, mag, amp, _ = attention64_over(q[r0:r0 + r], dequant(k, ks, tables[i], n), dequant(v, vs, tables[i], n), scale, window)
        assert (got[r0:r0 + r].double().cpu() - out).abs().le(attention_bound(out, mag, amp, q.shape[2])).all()
        r0 += r


def _put(cache, scales, block, values):
    """A block's values [16, hkv, d], rounded by its own scales."""
    s = power_scale(values.abs().amax((0, 2)))
    codes = (values / s[None, :, None]).float().clamp(-448, 448).to(FP8)
    cache.view(torch.uint8)[block] = codes.view(torch.uint8).to(cache.device)
    scales[block] = s.float().to(scales.device)


LOUD = [  # d, hkv, g, length, rows, window, page of the loud token, its place there
    (128, 2, 4, 300, 1, 0, 7, 3),
    (128, 2, 4, 300, 1, 0, 0, 0),
    (128, 2, 4, 300, 1, 0, 18, 5),                        # the newest page
    (64, 1, 12, 1000, 1, 0, 30, 15),
    (256, 1, 8, 700, 1, 0, 20, 9),
    (128, 1, 4, 200, 1, 100, 6, 2),                       # outside of the window, its neighbours are not
    (128, 2, 4, 300, 40, 0, 7, 3),
    (128, 2, 4, 300, 40, 0, 0, 1),
    (128, 2, 4, 300, 300, 0, 9, 14),                      # behind most rows
    (128, 2, 4, 300, 200, 0, 18, 11),                     # the newest token of all
    (64, 2, 3, 400, 150, 0, 12, 0),
    (64, 2, 3, 400, 150, 60, 16, 7),
    (256, 2, 8, 300, 40, 0, 3, 8),
    (256, 1, 4, 500, 300, 0, 20, 2),
    (256, 1, 4, 2100, 16, 0, 60, 2),
    (128, 1, 4, 4000, 30, 0, 100, 6),
]


@pytest.mark.parametrize("ratio", [16, 20, 26, 40])
@pytest.mark.parametrize("weight", ["none", "some"])
@pytest.mark.parametrize("d,hkv,g,n,r,window,page,place", LOUD)
def test_a_loud_token_beside_quiet_ones(d, hkv, g, n, r, window, page, place, weight, ratio):
    """One token's values are 2^ratio times all others'.  It has no weight to speak of, or one of about 2^-ratio, with which it is a good part of
    the output."""
    gen = torch.Generator().manual_seed(n + page)
    tables, nb = tables_for([n], gen, DEV)
    k, v, ks, vs = make_cache(nb, hkv, d, gen, DEV, spread=1)
    scale = d ** -0.5
    k.view(torch.uint8)[..., 0] = 0                        # channel 0 is that token's alone
    block = int(tables[0, page])
    keys, values = dequant(k, ks, tables[0, page:page + 1], BS), dequant(v, vs, tables[0, page:page + 1], BS)
    keys[place, :, 0] = -(150.0 if weight == "none" else ratio) / (4.0 * scale * 1.4427)
    values[place] *= 2.0 ** ratio
    _put(k, ks, block, keys)
    _put(v, vs, block, values)
    q = torch.randn(r, hkv * g, d, generator=gen) * 0.5
    q[..., 0] = 4.0
    _check(q.to(torch.bfloat16).to(DEV), k, v, ks, vs, tables, [n], [r], scale, window)


@pytest.mark.parametrize("spread", [12, 28])
@pytest.mark.parametrize("d,hkv,g,lens,rows,window", [
    (128, 4, 4, [300, 77, 1200], [1, 1, 1], 0), (64, 2, 16, [500, 31], [1, 1], 40), (256, 2, 5, [260, 700], [1, 1], 0),
    (128, 2, 4, [300, 129], [300, 40], 0), (64, 4, 3, [513], [200], 100), (256, 2, 8, [530, 70], [17, 70], 0), (128, 1, 8, [3000], [20], 0)])
def test_scales_all_over_the_place(d, hkv, g, lens, rows, window, spread):
    gen = torch.Generator().manual_seed(d + spread)
    tables, nb = tables_for(lens, gen, DEV)
    k, v, ks, vs = make_cache(nb, hkv, d, gen, DEV, spread=1)
    vs *= torch.exp2(torch.randint(-spread, spread + 1, (nb, hkv), generator=gen).float()).to(DEV)
    q = torch.randn(sum(rows), hkv * g, d, generator=gen).to(torch.bfloat16).to(DEV)
    _check(q, k, v, ks, vs, tables, lens, rows, d ** -0.5, window)


# ----------------------------------------------------------------------------- one batch on several streams, and with other lengths
def test_a_batch_is_used_on_a_second_stream_at_once():
    gen = torch.Generator().manual_seed(21)
    lens, rows = [900, 500], [900, 300]
    tables, nb = tables_for(lens, gen, DEV)
    k, v, ks, vs = make_cache(nb, 4, 128, gen, DEV)
    q = torch.randn(sum(rows), 16, 128, generator=gen).to(torch.bfloat16).to(DEV)

    def call(batch):
        w = torch.zeros(2, 4, 900, device=DEV)
        return ops.paged_attention(q, k, v, batch, 0.09, ks, vs, weights=w), w
    want = call(batch_of(lens, rows, tables))
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        batch, got = batch_of(lens, rows, tables), []
        torch.cuda.synchronize()
        for s in streams:                                  # fresh: the first call's lists may still be on their way
            with torch.cuda.stream(s):
                got.append(call(batch))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_a_batch_whose_sequences_grew():
    gen = torch.Generator().manual_seed(22)
    tables, nb = tables_for([400], gen, DEV)
    k, v, ks, vs = make_cache(nb, 2, 64, gen, DEV)
    q = torch.randn(30, 4, 64, generator=gen).to(torch.bfloat16).to(DEV)
    batch = batch_of([200], [30], tables)
    for n in (200, 390):
        batch.seq_lens.fill_(n)
        batch.seq_lens_host[0] = batch.max_seq_len = n
        w = torch.zeros(1, 2, 400, device=DEV)
        got = ops.paged_attention(q, k, v, batch, 0.125, ks, vs, weights=w)
        out, mag, amp, sums = attention64_over(q, dequant(k, ks, tables[0], n), dequant(v, vs, tables[0], n), 0.125)
        assert (got.double().cpu() - out).abs().le(attention_bound(out, mag, amp, 64)).all()
        rel = 4 * 12 * 2.0 ** -23 * (float(amp.max()) + 2.0) + 2.0 ** -20
        assert (w[0, :, :n].double().cpu() - sums).abs().le(rel * sums + 4 * 2.0 ** -23 * sums).all()


def test_prompt_rows_with_weights_in_a_graph():
    """Captured behind a first call on another stream; the batch then goes on with other lengths while the graph lives."""
    gen = torch.Generator().manual_seed(23)
    tables, nb = tables_for([300, 90], gen, DEV, extra_cols=4)
    k, v, ks, vs = make_cache(nb, 2, 128, gen, DEV)
    lens, rows = [300, 90], [40, 90]
    q = torch.randn(130, 8, 128, generator=gen).to(torch.bfloat16).to(DEV)
    batch = batch_of(lens, rows, tables)
    w = torch.zeros(2, 2, 320, device=DEV)
    call = lambda: ops.paged_attention(q, k, v, batch, 0.09, ks, vs, weights=w)
    want = call().clone(), w.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    batch.seq_lens_host[0] = 290                           # other lists from here on
    for _ in range(3):
        w.zero_()
        call()
    junk = [torch.full((2, n), 1 << 20, dtype=torch.int32, device=DEV) for n in range(1, 20)]
    w.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want[0]) and torch.equal(w, want[1]) and len(junk) == 19


# ----------------------------------------------------------------------------- softmax scales at their ends
@pytest.mark.parametrize("scale", [2.0 ** -60, 2.0 ** -30, 2.0 ** 4])
@pytest.mark.parametrize("d,lens,rows,window", [(128, [300, 50], [1, 1], 0), (128, [300, 50], [200, 50], 0), (64, [90], [90], 20), (256, [200, 40], [70, 1], 0)])
def test_softmax_scales_at_their_ends(d, lens, rows, window, scale):
    gen = torch.Generator().manual_seed(d)
    tables, nb = tables_for(lens, gen, DEV)
    k, v, ks, vs = make_cache(nb, 2, d, gen, DEV, spread=1)
    k.view(torch.uint8)[int(tables[0, 1])] = 0             # keys of nothing: the smallest scale
    ks[int(tables[0, 1])] = 2.0 ** -60
    q = torch.randn(sum(rows), 8, d, generator=gen).to(torch.bfloat16).to(DEV)
    _check(q, k, v, ks, vs, tables, lens, rows, scale, window)


# ----------------------------------------------------------------------------- sums much wider than the sequences
def test_scratch_goes_by_the_sequences_not_by_the_width_of_the_sums():
    gen = torch.Generator().manual_seed(31)
    lens = [100, 37, 60, 1]
    tables, nb = tables_for(lens, gen, DEV)
    k, v, ks, vs = make_cache(nb, 8, 64, gen, DEV)
    q = torch.randn(4, 32, 64, generator=gen).to(torch.bfloat16).to(DEV)
    call = lambda w: ops.paged_attention(q, k, v, batch_of(lens, [1] * 4, tables), 0.125, ks, vs, weights=w)
    narrow, wide = torch.zeros(4, 8, 100, device=DEV), torch.zeros(4, 8, 1 << 18, device=DEV)
    want = call(narrow)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = call(wide)
    # outputs, pieces and the scores of 4 x 8 x 100 x 4 heads: all below 8 MB; by the width the scores alone took 134 MB
    assert torch.cuda.max_memory_allocated() - before < 8 << 20
    assert torch.equal(got, want) and torch.equal(wide[..., :100], narrow) and not wide[..., 100:].any()


# ----------------------------------------------------------------------------- shares of the keys, empty ones among them
@pytest.mark.parametrize("d,hkv,g,lens,rows,window", [
    (128, 2, 4, [9000, 32], [1, 32], 0), (64, 1, 4, [20000, 3, 700], [1, 3, 20], 0), (256, 2, 4, [8000, 40], [1, 17], 0),
    (128, 1, 4, [6000, 20, 300], [30, 20, 10], 0), (64, 1, 8, [5000, 9], [16, 9], 1500), (256, 1, 8, [7000, 12], [10, 12], 0)])
def test_short_prompts_beside_long_sequences(d, hkv, g, lens, rows, window):
    check_attention(d, hkv, g, lens, rows, window, True, smallest=window > 0)
    torch.empty(1 << 26, device=DEV).fill_(float("nan"))    # what a workspace may hold
    check_attention(d, hkv, g, lens, rows, window, True, smallest=window > 0)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 40])
@pytest.mark.parametrize("d,lens,rows", [(128, [300, 200], [1, 200]), (64, [400], [100]), (256, [150], [90])])
def test_windows_longer_than_everything(d, lens, rows, window):
    gen = torch.Generator().manual_seed(d)
    tables, nb = tables_for(lens, gen, DEV)
    k, v, ks, vs = make_cache(nb, 2, d, gen, DEV)
    q = torch.randn(sum(rows), 8, d, generator=gen).to(torch.bfloat16).to(DEV)
    out = []
    for w in (None, window):
        sums = torch.zeros(len(lens), 2, max(lens), device=DEV)
        out.append((ops.paged_attention(q, k, v, batch_of(lens, rows, tables), d ** -0.5, ks, vs, w, weights=sums), sums))
    assert all(torch.equal(a, b) for a, b in zip(*out)) and out[0][1].sum() > 0


# ----------------------------------------------------------------------------- eviction
def test_eviction_takes_minus_infinity_before_nan():
    gen = torch.Generator().manual_seed(6)
    tables, nb = tables_for([60], gen, DEV)
    to, spare = tables_for([40], gen, DEV)
    k, v, ks, vs = make_cache(nb + spare, 2, 64, gen, DEV)
    w = torch.rand(1, 2, 60, generator=gen)
    w[..., ::3] = float("nan")
    w[..., 1::3] = float("-inf")
    for keep in (10, 30, 40):
        kept = ops.kv_evict(k, v, ks, vs, tables, torch.tensor([60], dtype=torch.int32, device=DEV), w.to(DEV), keep, to + nb, sink=1, recent=2)[1]
        for h in range(2):
            mid = sorted(range(1, 58), key=lambda j: (w[0, h, j] != w[0, h, j], -float(w[0, h, j].nan_to_num(0.0, neginf=-1.0)), j))
            assert kept[0, h].tolist() == sorted([0, 58, 59] + mid[:keep - 3])


# ----------------------------------------------------------------------------- queries at the ends of their type
@pytest.mark.parametrize("power,scale,key", [(116, 2.0 ** -60, -60), (-120, 2.0 ** 60, 58), (-126, 2.0 ** 60, 60), (90, 2.0 ** -45, -45)])
@pytest.mark.parametrize("d,lens,rows", [(128, [200, 33], [1, 1]), (64, [70], [1]), (256, [100], [1]), (128, [150], [40]), (256, [150], [40])])
def test_queries_of_any_size(d, lens, rows, power, scale, key):
    gen = torch.Generator().manual_seed(d + rows[0])
    tables, nb = tables_for(lens, gen, DEV)
    k, v, ks, vs = make_cache(nb, 2, d, gen, DEV, spread=1)
    for i in range(nb):
        k.view(torch.uint8)[i] = (torch.randn(BS, 2, d, generator=gen) * 0.5).to(FP8).view(torch.uint8).to(DEV)
    ks.fill_(2.0 ** key)
    q = (torch.randn(sum(rows), 8, d, generator=gen) * 2.0 ** power).to(torch.bfloat16).to(DEV)
    _check(q, k, v, ks, vs, tables, lens, rows, scale)


@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
@pytest.mark.parametrize("hkv,lens,keep,sink,recent", [
    (80, [9000], 50, 2, 3),                                # a block a head, more tokens than its registers hold
    (5, [9001, 8200, 20] * 6, 20, 0, 1),
    (40, [18011], 300, 1, 0),                              # two blocks a head
    (1, [80000], 4096, 16, 512),                           # eight
])
def test_evict_of_more_tokens_than_registers_hold(hkv, lens, keep, sink, recent, kind):
    gen = torch.Generator().manual_seed(keep)
    tables, nb = tables_for(lens, gen, DEV)
    to, spare = tables_for([min(n, keep) for n in lens], gen, DEV)
    k, v, ks, vs = make_cache(nb + spare, hkv, 64, gen, DEV)
    w = torch.rand(len(lens), hkv, max(lens), generator=gen)
    if kind == "ties":
        w = (w * 4).floor() / 4
    elif kind == "odd":
        w = torch.where(w < 0.2, torch.full_like(w, float("nan")), torch.where(w < 0.4, torch.full_like(w, float("inf")), w - 0.7))
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    new, kept, out_w = ops.kv_evict(k, v, ks, vs, tables, n, w.to(DEV), keep, to + nb, sink=sink, recent=recent)
    assert new.tolist() == [min(x, keep) for x in lens]
    kept, out_w = kept.cpu(), out_w.cpu()
    heavy = torch.where(w.isnan(), torch.full_like(w, float("-inf")), w).numpy()
    for i, m in enumerate(lens):
        for h in range(hkv):
            pos = np.arange(min(m, keep))
            if m > keep:
                mid = np.arange(sink, m - recent)
                best = mid[np.lexsort((mid, -heavy[i, h, mid]))][:keep - sink - recent]
                pos = np.sort(np.concatenate([np.arange(sink), best, np.arange(m - recent, m)]))
            assert kept[i, h, :len(pos)].tolist() == pos.tolist() and (kept[i, h, len(pos):] == -1).all()
            assert torch.equal(out_w[i, h, :len(pos)].view(torch.int32), w[i, h, torch.from_numpy(pos)].view(torch.int32))
        was, now = dequant(v, vs, tables[i], m)[:, 0], dequant(v, vs, to[i] + nb, min(m, keep))[:, 0]
        pages = torch.nn.functional.pad(was[kept[i, 0, :min(m, keep)].long()], (0, 0, 0, -min(m, keep) % BS)).view(-1, BS, 64)
        scale = power_scale(pages.abs().amax((1, 2)))[:, None, None]
        assert torch.equal(now, (nearest_e4m3(pages / scale) * scale).view(-1, 64)[:min(m, keep)])


# ----------------------------------------------------------------------------- writing steps of thousands of rows
@pytest.mark.parametrize("d,hkv,g,rot,norm,plus_one,lens,rows", [
    (64, 3, 2, 32, True, False, [40, 17, 1, 2500, 190], [1, 1, 1, 2100, 187]),         # single rows before prompts that begin inside a page
    (128, 1, 1, 128, False, False, [2041, 700], [2036, 13]),
    (256, 5, 1, 64, True, True, [16, 2200], [1, 2187]),
    (128, 2, 3, 0, False, False, [23] * 100, [21] * 100),                               # every run crosses a block's rows
    (64, 1, 4, 64, False, False, [7] * 300, [7] * 300),                                 # several runs in a block's rows
    (128, 9, 1, 16, True, False, [600], [520]), (64, 7, 2, 64, False, False, [2050], [2047]),      # on both sides of the plans' borders
    (64, 7, 2, 64, False, False, [2050], [2048]), (128, 3, 1, 128, False, False, [515], [512]), (128, 3, 1, 128, False, False, [515], [513]),
])
def test_writes_of_many_rows(d, hkv, g, rot, norm, plus_one, lens, rows):
    base.test_write_sets_and_raises_block_scales(d, hkv, g, rot, norm, plus_one, lens, rows)


@pytest.mark.parametrize("d,hkv,g,lens,rows,window", [
    (128, 2, 4, [300, 77], [1, 1], 0), (64, 2, 16, [500], [1], 40), (256, 2, 5, [260], [1], 0),
    (128, 2, 4, [300, 129], [300, 40], 0), (256, 2, 8, [530, 70], [17, 70], 0), (128, 1, 8, [3000], [20], 0)])
def test_weights_do_not_depend_on_the_values_scales(d, hkv, g, lens, rows, window):
    gen = torch.Generator().manual_seed(d)
    tables, nb = tables_for(lens, gen, DEV)
    k, v, ks, vs = make_cache(nb, hkv, d, gen, DEV, spread=1)
    vs *= torch.exp2(torch.randint(-28, 29, (nb, hkv), generator=gen).float()).to(DEV)
    q = torch.randn(sum(rows), hkv * g, d, generator=gen).to(torch.bfloat16).to(DEV)
    w = torch.zeros(len(lens), hkv, max(lens), device=DEV)
    ops.paged_attention(q, k, v, batch_of(lens, rows, tables), d ** -0.5, ks, vs, window or None, weights=w)
    r0 = 0
    for i, (n, r) in enumerate(zip(lens, rows)):
        _, _, amp, sums = attention64_over(q[r0:r0 + r], dequant(k, ks, tables[i], n), dequant(v, vs, tables[i], n), d ** -0.5, window)
        # scores and sums in fp32: the exponents s + ev - M and s - M are up to 100 larger than the scores
        rel = 4 * (d / 16 + 8) * 2.0 ** -23 * (float(amp.max()) + 102.0) + 2.0 ** -20 + (r * g / 32 + 8) * 2.0 ** -23
        assert (w[i, :, :n].double().cpu() - sums).abs().le(rel * sums + 1e-37).all() and not w[i, :, n:].any()
        r0 += r

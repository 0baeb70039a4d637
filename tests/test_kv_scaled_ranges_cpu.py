"""The block-scaled FP8 cache without a GPU, at the ends of what its calls allow."""
import ctypes
import pathlib
import re
import warnings

import pytest
import torch

from atlas_b200 import ops
from atlas_b200.config import tiny_deepseek, tiny_dense
from atlas_b200.ops import checked, cuda as K, cuda_scaled as CS
from kv_scaled_cases import BS, attention64_over, attention_bound, dequant, make_cache, tables_for
from test_kv_scaled_engine_cpu import engine
from test_kv_scaled_cpu import attend, batch_of, parts, write

CSRC = pathlib.Path(__file__).resolve().parent.parent / "atlas_b200" / "csrc"


def _kernels(text):
    for m in re.finditer(r"__global__[^;{]*\{", text):
        end = text.find("\n}\n", m.end())
        yield text[m.start():m.end()].split("(")[-2].split()[-1], text[m.end():end]


@pytest.mark.parametrize("name", ["attention_scaled_tc.cu", "kv_scaled.cu", "moe.cu"])
def test_a_cluster_meets_before_it_reaches_into_shared_memory(name):
    """Another CTA's shared memory is there only once that CTA has started, which a barrier of the cluster says."""
    seen = 0
    for _, body in _kernels((CSRC / name).read_text()):
        far = re.search(r"cluster_map_shared|ld_cluster|st_cluster", body)
        if far:
            seen += 1
            assert "cluster_sync_all();" in body[:far.start()]
    assert seen


def test_blocks_outside_of_the_pool_are_skipped():
    gen = torch.Generator().manual_seed(4)
    lens, rows = [40, 33, 30], [1, 20, 30]
    tables, nb = tables_for(lens, gen, "cpu")
    k, v, ks, vs = make_cache(nb, 2, 64, gen, "cpu", kernel_layout=False)
    kk = [dequant(k, ks, t, n) for t, n in zip(tables, lens)]
    vv = [dequant(v, vs, t, n) for t, n in zip(tables, lens)]
    there = [torch.ones(n, dtype=torch.bool) for n in lens]
    for i, page, entry in ((0, 1, -1), (1, 0, nb), (2, 0, -9)):                     # rows of the last sequence's first block see nothing
        tables[i, page] = entry
        there[i][page * BS:(page + 1) * BS] = False
    q = torch.randn(sum(rows), 4, 64, generator=gen).to(torch.bfloat16)
    w = torch.zeros(3, 2, 40)
    got = ops.paged_attention(q, k, v, batch_of(lens, rows, tables), 0.125, ks, vs, weights=w)
    n = torch.tensor(lens, dtype=torch.int32)
    read = ops.kv_read(k, v, tables, n, 40, ks, vs)
    r0 = 0
    for i, (m, r) in enumerate(zip(lens, rows)):
        out, mag, amp, sums = attention64_over(q[r0:r0 + r], kk[i], vv[i], 0.125, 0, there[i])
        assert (got[r0:r0 + r].double() - out).abs().le(attention_bound(out, mag, amp, 64)).all()
        tol = 4 * 72 * 2.0 ** -23 * (float(amp.max()) + 2.0) + 2.0 ** -20          # as an exponent: fp32 steps of a score, twice
        assert (w[i, :, :m].double() - sums).abs().le(tol * sums).all()
        for x, want in zip(read, (kk, vv)):
            assert torch.equal(x[i, :m].double(), want[i] * there[i][:, None, None])
        r0 += r
    old = k.view(torch.uint8).clone(), ks.clone()
    x = torch.ones(2, 2, 64, dtype=torch.bfloat16)
    ops.qk_norm_rope_kv_write(x, x, x, None, None, 0, k, v, torch.tensor([nb * BS, -3], dtype=torch.int32), ks, vs)
    assert torch.equal(k.view(torch.uint8), old[0]) and torch.equal(ks, old[1])


# ----------------------------------------------------------------------------- lists of a step
class Lists:
    """``step_list`` with streams, captures and uploads of the test's making."""

    def __init__(self, monkeypatch):
        self.place, self.uploads = (1, False), 0
        monkeypatch.setattr(K, "_list_place", lambda device: self.place)
        monkeypatch.setattr(K, "_upload", self.upload)

    def upload(self, rows, device):
        self.uploads += 1
        return torch.tensor(rows, dtype=torch.int32), None


def test_lists_of_a_step_follow_its_lengths_and_streams(monkeypatch):
    lists = Lists(monkeypatch)
    tables = torch.zeros(3, 40, dtype=torch.int32)
    b = batch_of([5, 300, 200], [1, 40, 200], tables)
    keys = lambda: CS._weigh_tiles(b, b.num_decodes, torch.device("cpu"))
    tiles = lambda tok: K._tc_tiles(tables, b, b.num_decodes, tok)
    first = keys()
    assert first[1] == 3 + 2 and keys()[0] is first[0] and lists.uploads == 1
    assert tiles(32)[1] == 2 + 7 and tiles(64)[1] == 1 + 4 and tiles(32)[1] == 9 and lists.uploads == 3      # of both sizes at once
    lists.place = (2, False)                                                   # a stream that the upload is not ordered with
    other = keys()
    assert other[0] is not first[0] and torch.equal(other[0], first[0]) and lists.uploads == 4
    lists.place = (1, False)
    assert keys()[0] is first[0]
    b.seq_lens_host[1] = 500                                                   # the sequence has grown
    grown = keys()
    assert grown[1] == 4 + 2 and sorted(grown[0][1][grown[0][0] == 1].tolist()) == [0, 128, 256, 384]
    b.query_lens_host[2] = 10
    assert tiles(32)[1] == 2 + 1


def test_what_a_graph_was_captured_with_stays(monkeypatch):
    lists = Lists(monkeypatch)
    b = batch_of([300], [40], torch.zeros(1, 40, dtype=torch.int32))
    keys = lambda: CS._weigh_tiles(b, b.num_decodes, torch.device("cpu"))
    warm = keys()[0]
    lists.place = (7, True)
    assert keys()[0] is warm and lists.uploads == 1                            # nothing uploaded inside the graph
    lists.place = (1, False)
    b.seq_lens_host[0] = 301
    assert keys()[0] is not warm
    assert any(t is warm for e in b._captured_lists for t in e)


@pytest.mark.parametrize("scale", [0.0, -0.125, float("nan"), float("inf"), 2.0 ** -61, 2.0 ** 61])
def test_softmax_scales_that_are_refused(scale):
    k, v, ks, vs = parts()
    for rows in ([1], [3]):
        b = batch_of([20], rows, torch.zeros(1, 2, dtype=torch.int32))
        q = torch.ones(rows[0], 4, 64, dtype=torch.bfloat16)
        with pytest.raises(K.KernelError, match="softmax scale"):
            CS.paged_attention(q, k, v, b, scale, ks, vs)
        with pytest.raises(ValueError, match="softmax scale"):
            ops.paged_attention(q, k, v, b, scale, ks, vs)


def test_shares_of_the_keys_go_by_the_prompts():
    assert CS.key_shares([], 0, 0, 148) == 1
    assert CS.key_shares([32], 8, 0, 148) == 1                                 # beside any number of long single tokens
    assert CS.key_shares([65000, 100], 8, 0, 148) == 18
    assert CS.key_shares([4096], 8, 0, 148) == 8                               # at least 512 tokens each
    assert CS.key_shares([65000], 8, 2000, 148) == 4
    assert CS.key_shares([65000], 200, 0, 148) == 1


class Records:
    """The records of the attention's calls, as far as they go without a GPU."""

    def __init__(self, monkeypatch):
        self.seen = {}
        Lists(monkeypatch)
        monkeypatch.setattr(CS, "_call", lambda name, record, what: self.seen.update({name: record}))
        monkeypatch.setattr(CS, "_place", lambda t: (CS._HERE, 0, 0))
        monkeypatch.setitem(K._num_sms, 0, 148)
        monkeypatch.setitem(K._status_ptr, 0, 0)

    def decode(self, field):
        return CS._DECODE.unpack(self.seen["atlas_attn_scaled_decode"])[field]

    def chunk(self, field):
        return CS._CHUNK.unpack(self.seen["atlas_attn_scaled_chunk"])[field]


def test_short_prompts_beside_a_long_single_token_are_not_cut(monkeypatch):
    records = Records(monkeypatch)
    k, v, ks, vs = parts()
    for lens, rows, want in (([40000, 32], [1, 32], 1), ([40000, 9000], [1, 32], 17)):
        b = batch_of(lens, rows, torch.zeros(2, 2500, dtype=torch.int32))
        CS.paged_attention(torch.zeros(33, 4, 64, dtype=torch.bfloat16), k, v, b, 0.125, ks, vs)
        assert records.chunk(27) == want


def test_windows_reach_no_further_than_the_tables(monkeypatch):
    records = Records(monkeypatch)
    k, v, ks, vs = parts()
    b = batch_of([30, 20], [1, 7], torch.zeros(2, 2, dtype=torch.int32))
    for window, want in ((None, 0), (5, 5), (32, 32), (33, 32), (2 ** 31 - 1, 32), (2 ** 40, 32)):
        CS.paged_attention(torch.zeros(8, 4, 64, dtype=torch.bfloat16), k, v, b, 0.125, ks, vs, window)
        assert records.decode(21) == records.chunk(24) == want


# ----------------------------------------------------------------------------- refusals
def test_what_is_written_has_places_of_its_own():
    k, v, ks, vs = parts()
    one = torch.ones(1, 1)
    good = torch.ones(4, 5)[:, ::2][:, :2], torch.ones(2, 4).t()               # strides of their own kind, but apart
    for scales in ((one.expand(4, 2), vs), (ks, one.expand(4, 2)), (ks, ks), (torch.ones(4, 1).expand(4, 2), vs),
                   (torch.ones(8).as_strided((4, 2), (1, 1)), vs), (torch.ones(8).as_strided((4, 2), (1, 2)), vs)):
        with pytest.raises(K.KernelError, match="places of their own"):
            write(k, v, *scales)
        with pytest.raises(K.KernelError, match="places of their own"):
            CS.kv_evict(k, v, *scales, torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros(1, 2, 9), 4,
                        torch.zeros(1, 2, dtype=torch.int32), 0, 0)
    with pytest.raises(K.KernelError, match="GPU"):                             # past the checks
        write(k, v, *good)
    for w in (torch.zeros(1, 2, 32).expand(2, 2, 32), torch.zeros(2, 1, 32).expand(2, 2, 32), torch.zeros(200).as_strided((2, 2, 32), (40, 20, 1))):
        with pytest.raises(K.KernelError, match="of its own"):
            attend(k, v, ks, vs, weights=w)
    with pytest.raises(K.KernelError, match="GPU"):
        attend(k, v, ks, vs, weights=torch.zeros(2, 3, 40)[:, 1:, 3:])


def test_no_heads_are_refused():
    k, v, ks, vs = parts()
    with pytest.raises(K.KernelError, match="0 query heads"):
        attend(k, v, ks, vs, q=torch.zeros(2, 0, 64, dtype=torch.bfloat16))
    for call in (attend, write):
        with pytest.raises(K.KernelError, match="at least one head"):
            call(*parts(hkv=0))


def test_entry_points_refuse_what_would_divide_by_zero():
    """Straight at the library: these returns come before anything is launched."""
    if not pathlib.Path(K.LIB_PATH).exists():
        pytest.skip("the kernels are not built")
    lib = K.lib()
    for name, record, hq in (("atlas_attn_scaled_decode", CS._DECODE, 18), ("atlas_attn_scaled_chunk", CS._CHUNK, 21)):
        f = getattr(lib, name)
        f.argtypes = [ctypes.c_char_p]
        n = len(record.unpack(bytes(record.size)))
        real = next(i for i, x in enumerate(record.unpack(bytes(record.size))) if isinstance(x, float))
        for heads in ((0, 1), (1, 2), (129, 1)):
            a = [0] * n
            a[real] = 0.125
            a[17] = a[19] = 1                                                  # one sequence, one tile
            a[hq], a[hq + 1], a[hq + 2] = heads + (64,)
            assert f(record.pack(*a)) == -1


def test_eviction_takes_minus_infinity_before_nan():
    gen = torch.Generator().manual_seed(6)
    tables, nb = tables_for([60], gen, "cpu")
    to, spare = tables_for([40], gen, "cpu")
    k, v, ks, vs = make_cache(nb + spare, 2, 64, gen, "cpu", kernel_layout=False)
    w = torch.rand(1, 2, 60, generator=gen)
    w[..., ::3] = float("nan")
    w[..., 1::3] = float("-inf")
    for keep in (10, 30, 40):
        kept = ops.kv_evict(k, v, ks, vs, tables, torch.tensor([60], dtype=torch.int32), w, keep, to + nb, sink=1, recent=2)[1]
        for h in range(2):
            mid = sorted(range(1, 58), key=lambda j: (w[0, h, j] != w[0, h, j], -float(w[0, h, j].nan_to_num(0.0, neginf=-1.0)), j))
            assert kept[0, h].tolist() == sorted([0, 58, 59] + mid[:keep - 3])


def test_attention_wants_a_row_for_every_new_token():
    parts_ = parts()
    for rows, T in (((1, 5), 5), ((5, 5), 9), ((20, 3), 22)):
        with pytest.raises(K.KernelError, match="query rows for"):
            attend(*parts_, rows=rows, q=torch.zeros(T, 4, 64, dtype=torch.bfloat16))
    k, v, ks, vs = parts_
    b = batch_of([20, 5], [1, 5], torch.zeros(2, 2, dtype=torch.int32))
    b.query_lens_host = []
    with pytest.raises(K.KernelError, match="host lengths"):
        CS.paged_attention(torch.zeros(6, 4, 64, dtype=torch.bfloat16), k, v, b, 0.1, ks, vs)


def test_eviction_wants_a_weight_for_every_token():
    k, v, ks, vs = parts()
    t, n = torch.zeros(1, 2, dtype=torch.int32), torch.tensor([20], dtype=torch.int32)
    to = torch.ones(1, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="weights of 19 tokens"):
        ops.kv_evict(k, v, ks, vs, t, n, torch.zeros(1, 2, 19), 17, to)
    with pytest.raises(checked.BoundsViolation):
        checked.evict(t, n, to, 4, 16, 17, 19)


# ----------------------------------------------------------------------------- the engine's option
@pytest.mark.parametrize("make, kw", [(tiny_deepseek, {}), (tiny_dense, {"block_size": 32}), (tiny_dense, {"sparse_attention_blocks": 8})])
def test_the_engine_says_where_block_scales_do_not_apply(make, kw):
    with pytest.warns(UserWarning, match="fp8_scaled"):
        assert not engine(make(), **kw).kv_block_scales


def test_the_engine_is_silent_where_they_do():
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert engine().kv_block_scales

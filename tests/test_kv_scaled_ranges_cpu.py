"""The block-scaled FP8 cache without a GPU, at the ends of what its calls allow."""
import pathlib
import re

import pytest
import torch

from atlas_b200 import ops
from kv_scaled_cases import BS, attention64_over, attention_bound, dequant, make_cache, tables_for
from test_kv_scaled_cpu import batch_of

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

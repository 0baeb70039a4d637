"""Engines whose FP8 cache has a scale per (block, head): chosen by ``kv_cache_dtype="fp8_scaled"``, kept by swapped sequences, and not
chosen where a layer cannot have it."""
import pytest
import torch

from atlas_b200 import ops
from atlas_b200.config import EngineConfig, tiny_deepseek, tiny_dense, tiny_hybrid
from atlas_b200.engine import LLMEngine
from atlas_b200.kv.host_tier import HostKVTier
from atlas_b200.models import build_model
from atlas_b200.models.batch import ForwardBatch
from atlas_b200.sampling import SamplingParams

FP8 = torch.float8_e4m3fn


def engine(cfg=None, **kw):
    kw = {"num_kv_blocks": 64, "max_num_seqs": 8, "kv_cache_dtype": "fp8_scaled", **kw}
    return LLMEngine(build_model(cfg or tiny_dense()).init_random(0), EngineConfig(**kw))


def prompts(n, length):
    g = torch.Generator().manual_seed(3)
    return [torch.randint(0, 1024, (length,), generator=g).tolist() for _ in range(n)]


@pytest.mark.parametrize("make", [tiny_dense, tiny_hybrid])
def test_every_attention_layer_has_scales_of_its_own(make):
    eng = engine(make())
    assert eng.kv_block_scales and eng.kv_dtype == FP8
    for l in eng.model.attention_layers():
        k, v, ks, vs = eng.cache.layer_kv(l)
        assert k.dtype == v.dtype == FP8
        assert ks.shape == vs.shape == (64, 2) and bool((ks == 1).all())
    out = eng.generate(prompts(3, 24), SamplingParams(max_tokens=6, ignore_eos=True))
    assert all(len(o.output_tokens) == 6 for o in out)
    for l in eng.model.attention_layers():
        ks = eng.cache.layer_kv(l)[2]
        used = ks[ks != 1]
        assert used.numel() and bool((torch.frexp(used)[0] == 0.5).all())


def test_a_cache_scaled_by_block_is_nearer_than_one_scale():
    """Keys 2^-9 of their size put most codes of a cache with scale 1 below e4m3's smallest normal number, 2^-6; scales of the blocks bring
    them back.  The logits of both are held against a cache in 32 bits.  The values' rounding, about the same in both, bounds what the keys'
    scales can save: with error energies V + K' and V + K all that follows from K' < K is that the first is the smaller."""
    cfg = tiny_dense()
    model = build_model(cfg).init_random(0)
    for l in model.layers:
        w = l.mixer.qkv.weight
        n = l.mixer.hq * l.mixer.d
        w[:n] *= 2.0 ** 9                                   # the scores stay as they are
        w[n:n + l.mixer.hkv * l.mixer.d] *= 2.0 ** -9
    toks = prompts(1, 40)[0]
    fb = ForwardBatch.build([toks], [0], [[2, 0, 1]], 16, all_logits=True)
    run = lambda **kw: model.compute_logits(model.forward(fb, model.alloc_cache(4, 16, **kw))).double()
    exact = run(kv_dtype=torch.float32)
    one, each = run(kv_dtype=FP8), run(kv_dtype=FP8, block_scales=True)
    assert (each - exact).square().mean() < (one - exact).square().mean()


@pytest.mark.parametrize("make, kw", [(tiny_deepseek, {}), (tiny_dense, {"block_size": 32}), (tiny_dense, {"sparse_attention_blocks": 8})])
def test_where_it_does_not_apply_the_cache_is_plain_fp8(make, kw):
    eng = engine(make(), **kw)
    assert not eng.kv_block_scales and eng.kv_dtype == FP8
    assert all(s == (1.0, 1.0) for s in eng.cache.kv_scales.values())


def test_layers_of_high_precision_keep_a_cache_without_scales():
    eng = engine(kv_high_precision_layers=(0,))
    assert eng.cache.kv_scales[0] == (1.0, 1.0) and isinstance(eng.cache.kv_scales[1][0], torch.Tensor)
    assert eng.cache.kv[0][0].dtype != FP8 and eng.cache.kv[1][0].dtype == FP8
    eng.generate(prompts(2, 20), SamplingParams(max_tokens=3, ignore_eos=True))


def test_swapped_sequences_resume_with_their_scales():
    sp = SamplingParams(max_tokens=40, ignore_eos=True)
    want = [o.output_tokens for o in engine(max_prefill_tokens=64).generate(prompts(4, 40), sp)]
    swap = engine(max_prefill_tokens=64, num_kv_blocks=14, swap_space_gb=0.01)
    assert [o.output_tokens for o in swap.generate(prompts(4, 40), sp)] == want
    assert swap.scheduler.num_swaps > 0 and swap.host_tier.blocks_in == swap.host_tier.blocks_out > 0


def test_a_record_of_the_host_tier_holds_a_block_and_its_scales():
    model = build_model(tiny_dense()).init_random(0)
    cache = model.alloc_cache(6, 16, FP8, block_scales=True)
    assert model.kv_bytes_per_block(16, FP8, block_scales=True) == 2 * 2 * 2 * (16 * 64 + 4)
    tier = HostKVTier(cache, 3)
    assert tier.record_bytes == model.kv_bytes_per_block(16, FP8, block_scales=True)
    model.forward(ForwardBatch.build([list(range(70))], [0], [[4, 1, 0, 2, 5]], 16), cache)
    bits = lambda l, b: [t[b].float().clone() for t in cache.layer_kv(l)]
    before = [[bits(l, b) for b in (1, 5)] for l in (0, 1)]
    tier.copy_out([1, 5], [2, 0])
    for l in (0, 1):
        for t in cache.layer_kv(l):
            t.zero_()
    tier.copy_in([2, 0], [3, 1])
    for l in (0, 1):
        for b, was in zip((3, 1), before[l]):
            assert all(torch.equal(a, x) for a, x in zip(bits(l, b), was))


def test_draft_head_beside_scaled_layers():
    eng = engine(tiny_hybrid(), speculative=True, num_drafts=2)
    assert eng.spec is not None and eng.cache.kv_scales[eng.model.mtp.layer_idx] == (1.0, 1.0)
    plain = engine(tiny_hybrid())
    sp = SamplingParams(max_tokens=12, ignore_eos=True)
    a, b = ([o.output_tokens for o in e.generate(prompts(3, 20), sp)] for e in (eng, plain))
    assert all(len(x) == 12 for x in a) and [x[0] for x in a] == [x[0] for x in b]


def test_fused_output_form_leaves_a_scaled_cache_to_plain_attention():
    ks, vs = ops.alloc_kv_scales(4, 2, "cpu")
    assert ops.paged_attention_fp8_out(torch.zeros(1, 4, 64), None, None, None, 1.0, ks, vs) is None

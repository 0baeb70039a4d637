"""Models and engines on the GPU whose FP8 cache has a scale per (block, head) (``kv_cache_dtype="fp8_scaled"``)."""
import pytest
import torch

from atlas_b200 import ops
from atlas_b200.config import EngineConfig, ModelConfig, QuantConfig
from atlas_b200.engine import LLMEngine
from atlas_b200.models import build_model
from atlas_b200.models.batch import ForwardBatch
from atlas_b200.sampling import SamplingParams

pytestmark = pytest.mark.gpu
DEV, FP8 = "cuda", torch.float8_e4m3fn


@pytest.fixture(scope="module")
def K():
    from atlas_b200.ops import cuda
    return cuda


def config(d=128, quant="fp8_block", **kw):
    kw = {"vocab_size": 4096, "hidden_size": 1024, "intermediate_size": 2048, "num_hidden_layers": 2, "num_attention_heads": 8,
          "num_key_value_heads": 2, "rope_theta": 5e5, **kw}
    return ModelConfig(model_type="llama", family="dense", head_dim=d, max_position_embeddings=2048, quant=QuantConfig(method=quant), **kw)


def prompts(lengths, seed=4):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 4096, (n,), generator=g).tolist() for n in lengths]


@pytest.mark.parametrize("d, extra", [(64, {}), (128, {"qk_norm": True}), (256, {}), (128, {"sliding_window": 32})])
def test_logits_of_kernels_beside_the_plain_forms(K, d, extra):
    """A prompt in two chunks and one decode step, by the kernels and by the plain forms.  Both round keys, values and layer outputs to the
    same types; the bounds are those of the model tests of the other cache types."""
    model = build_model(config(d, "none", **extra), device=DEV).init_random(0)
    toks, tables = prompts([49])[0], [[3, 1, 4, 0]]
    logits = []
    for force in (False, True):
        ops.FORCE_REFERENCE = force
        try:
            cache = model.alloc_cache(8, 16, FP8, block_scales=True)
            steps = ((toks[:30], 0), (toks[30:48], 30), (toks[48:], 48))
            batches = [ForwardBatch.build([t], [n], tables, 16, device=DEV, all_logits=True) for t, n in steps]
            logits.append(torch.cat([model.compute_logits(model.forward(b, cache)) for b in batches]).float())
        finally:
            ops.FORCE_REFERENCE = False
    torch.cuda.synchronize()
    assert K.check_status() == 0
    got, want = logits
    assert (got - want).square().mean().sqrt() < 8e-2 * want.square().mean().sqrt()
    assert (got.argmax(-1) == want.argmax(-1)).float().mean() > 0.85


def test_graphs_and_prefix_cache(K):
    model = build_model(config(), device=DEV).init_random(0)
    ask, sp = prompts([40 + 7 * i for i in range(6)]), SamplingParams(max_tokens=12, ignore_eos=True)
    make = lambda graphs: LLMEngine(model, EngineConfig(num_kv_blocks=256, max_num_seqs=8, max_seq_len=512, max_prefill_tokens=128,
                                                        use_cuda_graphs=graphs, kv_cache_dtype="fp8_scaled"))
    e1, e2 = make(True), make(False)
    assert e1.kv_block_scales and isinstance(e1.cache.kv_scales[0][0], torch.Tensor)
    a, b = e1.generate(ask, sp), e2.generate(ask, sp)
    torch.cuda.synchronize()
    assert K.check_status() == 0 and e1.runner.graph_replays > 0
    # a replay pads the batch, which moves the cuts between the pieces of its attention and with them some roundings
    assert sum(x.output_tokens == y.output_tokens for x, y in zip(a, b)) >= 4
    again = e1.generate(ask[:2], sp)
    assert again[0].cached_tokens >= 32
    assert [o.output_tokens for o in again] == [o.output_tokens for o in a[:2]]


def test_host_tier_swap(K):
    model = build_model(config(), device=DEV).init_random(0)
    ask, sp = prompts([40] * 4, seed=3), SamplingParams(max_tokens=40, ignore_eos=True)
    make = lambda **kw: LLMEngine(model, EngineConfig(max_num_seqs=8, max_seq_len=512, max_prefill_tokens=64, use_cuda_graphs=False,
                                                      kv_cache_dtype="fp8_scaled", **kw))
    want = [o.output_tokens for o in make(num_kv_blocks=64).generate(ask, sp)]
    e = make(num_kv_blocks=14, swap_space_gb=0.01)
    got = [o.output_tokens for o in e.generate(ask, sp)]
    torch.cuda.synchronize()
    assert K.check_status() == 0
    assert e.scheduler.num_swaps > 0 and e.host_tier.blocks_in == e.host_tier.blocks_out > 0
    assert sum(a == b for a, b in zip(got, want)) >= 3                       # other batches, other pieces of the attention


def test_host_tier_carries_the_scales(K):
    from atlas_b200.kv.host_tier import HostKVTier
    model = build_model(config(), device=DEV).init_random(0)
    cache = model.alloc_cache(6, 16, FP8, block_scales=True)
    tier = HostKVTier(cache, 3)
    model.forward(ForwardBatch.build([prompts([70])[0]], [0], [[4, 1, 0, 2, 5]], 16, device=DEV), cache)
    bits = lambda l, b: [t[b].contiguous().view(torch.uint8) for t in cache.layer_kv(l)]
    before = [[bits(l, b) for b in (1, 5)] for l in (0, 1)]
    for n in (2, 1):                                                         # the record of one block alone keeps its alignment
        tier.copy_out([1, 5][:n], [2, 0][:n])
        for l in (0, 1):
            for t in cache.layer_kv(l)[2:]:
                t[2:4].zero_()
        tier.copy_in([2, 0][:n], [3, 2][:n])
        torch.cuda.synchronize()
        for l in (0, 1):
            for b, was in zip((3, 2), before[l][:n]):
                assert all(torch.equal(a, x) for a, x in zip(bits(l, b), was))

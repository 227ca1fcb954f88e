"""The engine on a 4-bit K/V cache on a B200: kernels against the reference ops, graphs, forks."""

import pytest
import torch

from everserve_b200.engine import Engine, EngineConfig, SamplingParams
from everserve_b200.models.config import SMALL_LLAMA, TINY_LLAMA, TINY_QWEN, ModelConfig
from everserve_b200.ops import RefOps, ref

pytestmark = pytest.mark.gpu

# grouped heads of 128, as the 8B model's
D128 = ModelConfig(name="d128", vocab=1024, hidden=512, layers=2, heads=8, kv_heads=2, head_dim=128, intermediate=512,
                   rope_theta=5e5, rms_eps=1e-5, max_position=2048)


def _cfg(model, graphs=True, **kw):
    return EngineConfig(model, device="cuda", max_batch=8, max_model_len=1024, num_blocks=256, use_cuda_graphs=graphs,
                        kv_quant="int4", **kw)


@pytest.mark.parametrize("model,kw", [(TINY_LLAMA, {}), (TINY_QWEN, {}), (D128, {}), (D128, dict(kv_group=0, block_size=32))])
def test_forward_matches_reference(cuda, model, kw):
    eng = Engine(_cfg(model, False, **kw))
    worker = eng.executor.worker
    for p in ([3, 1, 4, 1, 5, 9, 2, 6], list(range(40, 177)), [9]):
        eng.add_request(p, SamplingParams(max_tokens=4))
    runner, m = worker.runner, worker.model
    inp = runner.prefill_input(eng.scheduler.schedule())
    logits_k = m.logits(inp, runner.caches)
    kops = m.ops
    m.ops = RefOps("cuda")
    try:
        caches_ref = [torch.zeros_like(c) for c in runner.caches]
        logits_r = m.logits(inp, caches_ref)
    finally:
        m.ops = kops
    torch.testing.assert_close(logits_k.float(), logits_r.float(), rtol=5e-2, atol=5e-2)
    bs = eng.cfg.block_size
    held = [ref.kv4_cache_values(c, m.d, bs) for c in (runner.caches[0], caches_ref[0])]
    torch.testing.assert_close(held[0], held[1], rtol=5e-2, atol=5e-2)
    assert kops.check_status() == 0


@pytest.mark.parametrize("model", [TINY_QWEN, D128, SMALL_LLAMA])
def test_graphs_multistep_and_async_match_eager(cuda, model):
    prompts = [[i, i + 1, i + 2, 7] * (4 * i + 1) for i in range(1, 6)]
    outs = []
    for graphs, ahead in ((False, False), (True, False), (True, True)):
        outs.append(Engine(_cfg(model, graphs, async_decode=ahead)).generate(prompts, max_tokens=12))
    assert outs[0] == outs[1] == outs[2]
    eng = Engine(_cfg(model))
    ids = [eng.add_request(p, SamplingParams(max_tokens=12)) for p in prompts]
    eng.step()
    eng.step()
    eng.decode_steps(8)
    while eng.has_work():
        eng.step()
    assert [eng.request(i).outputs for i in ids] == outs[0]


@pytest.mark.parametrize("kv", [None, "int4"])
def test_samples_are_their_seeds_own_runs(cuda, kv):
    """Completions forked from one prefill (full blocks shared, the last one copied) draw what the prompt
    with the same seed draws in the same batch of decode rows."""
    prompt = [(5 * i + 2) % 500 for i in range(75)]
    kw = dict(max_tokens=24, temperature=0.8, top_k=30)
    cfg = lambda: EngineConfig(D128, device="cuda", max_batch=4, max_model_len=512, num_blocks=64, kv_quant=kv)  # noqa: E731
    eng = Engine(cfg())
    got = eng.samples(prompt, 4, seed=5, **kw)
    assert eng.blocks.free_blocks == 64 and len({tuple(g) for g in got}) > 1
    assert eng.executor.worker.model.ops.check_status() == 0
    # decode from a copied or shared block is decode from the block itself
    twin = Engine(cfg())
    rid = twin.add_request(prompt, SamplingParams(max_tokens=30))
    for _ in range(6):
        twin.step()
    other = twin.fork(rid)
    while twin.has_work():
        twin.step()
    assert twin.request(rid).outputs == twin.request(other).outputs


@pytest.mark.parametrize("kv", [None, "int4"])
@pytest.mark.parametrize("plen", [64, 65, 75])
def test_forks_of_one_seed_agree(cuda, kv, plen):
    """Forks that read the common blocks together and their own copy of the last one draw the same from one seed, and
    others from another."""
    prompt = [(5 * i + 2) % 500 for i in range(plen)]
    cfg = lambda: EngineConfig(D128, device="cuda", max_batch=4, max_model_len=512, num_blocks=64, kv_quant=kv)  # noqa: E731
    eng = Engine(cfg())
    rid = eng.add_request(prompt, SamplingParams(max_tokens=20))
    eng.step()
    draw = lambda seed: SamplingParams(max_tokens=20, temperature=0.8, top_k=30, seed=seed)  # noqa: E731
    ids = [eng.fork(rid, draw(seed), keep=plen) for seed in (9, 9, 10)]
    while eng.has_work():
        eng.step()
    a, b, c = (eng.request(i).outputs for i in ids)
    assert len(a) == 20 and a == b and a != c and eng.blocks.free_blocks == 64
    assert eng.executor.worker.model.ops.check_status() == 0

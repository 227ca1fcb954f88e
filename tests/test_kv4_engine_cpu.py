"""The engine on a 4-bit K/V cache and forked requests, on the CPU's reference ops."""

import pytest
import torch

from everserve_b200.engine import Engine, EngineConfig, SamplingParams
from everserve_b200.engine.block_manager import BlockManager
from everserve_b200.models.config import LLAMA3_8B, TINY_LLAMA, TINY_MIXTRAL, TINY_QWEN
from everserve_b200.models.llama import DecoderLM


def _engine(model=TINY_LLAMA, **kw):
    args = dict(device="cpu", dtype=torch.float32, max_batch=4, max_model_len=256, num_blocks=64)
    args.update(kw)
    return Engine(EngineConfig(model, **args))


@pytest.mark.parametrize("model", [TINY_LLAMA, TINY_QWEN, TINY_MIXTRAL])
def test_generate_on_4_bits(model):
    """Decoding from the cache predicts what a prefill of the same tokens predicts."""
    prompt = [(7 * i + 3) % 500 for i in range(40)]
    eng = _engine(model, kv_quant="int4")
    assert eng.executor.worker.runner.caches[0].dtype == torch.uint8
    out = eng.generate([prompt, prompt[:9]], max_tokens=6)
    again = _engine(model, kv_quant="int4").generate([prompt + out[0][:-1]], max_tokens=1)
    assert again[0] == [out[0][-1]]


def test_memory_of_a_block():
    def model(**kw):
        return DecoderLM(LLAMA3_8B, "cpu", torch.bfloat16, layer_range=(0, 1), init="none", **kw)

    dense, int4, whole = (model(**kw).bytes_per_block(16) for kw in ({}, {"kv_quant": "int4"}, {"kv_quant": "int4", "kv_group": 0}))
    assert (dense, int4, whole) == (16 * 8 * 512, 16 * 8 * 144, 16 * 8 * 136)


def test_config_refused():
    for kw in (dict(kv_quant="int3"), dict(kv_quant="int4", kv_group=32)):
        with pytest.raises(ValueError):
            EngineConfig(TINY_LLAMA, device="cpu", **kw)
    with pytest.raises(ValueError):
        Engine(EngineConfig(TINY_LLAMA, device="cpu", dtype=torch.float32, num_blocks=8, kv_quant="int4"), connector=object())
    from everserve_b200.serving.executor import MultiprocExecutor

    with pytest.raises(ValueError):
        MultiprocExecutor(EngineConfig(TINY_LLAMA, device="cpu", kv_quant="int4"))


def test_store_refused_however_attached(monkeypatch):
    """A committed-KV store commits rows of the unquantized cache: no way of attaching one to a 4-bit cache, or to
    requests that hold blocks together, is open, and a refused engine loads nothing."""
    from everserve_b200.engine import engine as module
    from everserve_b200.plugin import register

    eng = _engine(kv_quant="int4")
    with pytest.raises(ValueError):
        register(eng, connector=object(), prepare=False)
    with pytest.raises(ValueError):
        eng.connector = object()
    assert eng.connector is None
    eng = _engine()
    rid = eng.add_request(list(range(1, 20)), SamplingParams(max_tokens=8))
    eng.step()
    twin = eng.fork(rid)
    with pytest.raises(ValueError):
        register(eng, connector=object(), prepare=False)
    while eng.has_work():
        eng.step()
    assert eng.request(twin).outputs == eng.request(rid).outputs
    store = object()
    register(eng, connector=store, prepare=False)
    assert eng.connector is store
    monkeypatch.setattr(module, "LocalExecutor", lambda cfg: pytest.fail("an executor was built"))
    with pytest.raises(ValueError):
        Engine(EngineConfig(TINY_LLAMA, device="cpu", dtype=torch.float32, num_blocks=8, kv_quant="int4"), connector=store)


def test_shared_blocks():
    bm = BlockManager(4, 16)
    a = []
    bm.grow(a, 33)
    b, c = bm.share(a[:2]), bm.share(a[:1])
    bm.free(a)
    assert bm.free_blocks == 2 and b == [0, 1]
    bm.free(b)
    assert bm.free_blocks == 3 and c == [0]
    bm.free(c)
    assert bm.free_blocks == 4
    d = []
    bm.grow(d, 64)
    assert d == [0, 1, 2, 3]


@pytest.mark.parametrize("kv", [None, "int4"])
@pytest.mark.parametrize("plen", [1, 16, 17, 31, 40])
def test_samples_are_their_seeds_own_runs(kv, plen):
    """Forked completions draw what the same prompt and seed draw by themselves."""
    prompt = [(5 * i + 2) % 500 for i in range(plen)]
    kw = dict(max_tokens=20, temperature=0.9, top_k=20)
    eng = _engine(kv_quant=kv)
    got = eng.samples(prompt, 3, seed=11, **kw)
    assert eng.blocks.free_blocks == 64
    alone = [_engine(kv_quant=kv).generate([prompt], seed=11 + i, **kw)[0] for i in range(3)]
    assert got == alone and got[0] != got[1]


class _Store:
    """A connector that watches."""

    def begin_step(self, plan, scheduler):
        pass

    end_step = begin_step

    def finished(self, req_id):
        pass


class _Apart:
    """An executor that runs plans and copies no blocks."""

    def __init__(self, inner):
        self.inner, self.num_blocks = inner, inner.num_blocks

    def execute(self, plan):
        return self.inner.execute(plan)

    def fetch(self, ids):
        return self.inner.fetch(ids)


@pytest.mark.parametrize("how", ["store", "executor", "one token", "small batch"])
def test_samples_where_not_all_are_forks(how):
    """Completions that cannot be forked prefill the prompt themselves; no request is left behind."""
    prompt = [(5 * i + 2) % 500 for i in range(19)]
    kw = dict(max_tokens=1 if how == "one token" else 6, temperature=0.9, top_k=20, seed=3)
    eng = _engine(max_batch=2 if how == "small batch" else 4)
    if how == "store":
        eng.connector = _Store()
    if how == "executor":
        eng.executor, eng.async_decode = _Apart(eng.executor), False
    got = eng.samples(prompt, 5, **kw)
    assert not eng.has_work() and eng.blocks.free_blocks == 64
    seed = kw.pop("seed")
    assert got == [_engine().generate([prompt], seed=seed + i, **kw)[0] for i in range(5)]


def test_fork_mid_way():
    """A fork of a request under way continues as the request does; one from an earlier token replays it;
    results the fork had to apply come with the next step."""
    eng = _engine()
    rid = eng.add_request([3, 1, 4, 1, 5, 9, 2, 6, 5, 3, 5, 8, 9, 7, 9, 3, 2, 3, 8], SamplingParams(max_tokens=24))
    seen = []
    for _ in range(8):
        seen += eng.step()
    twin = eng.fork(rid)
    back = eng.fork(rid, keep=21)
    while eng.has_work():
        seen += eng.step()
    out = eng.request(rid).outputs
    assert len(out) == 24 and eng.request(twin).outputs == out and eng.request(back).outputs == out
    assert [t for r, t, _ in seen if r == rid] == out
    assert eng.blocks.free_blocks == 64
    with pytest.raises(ValueError):
        eng.fork(rid)  # finished
    with pytest.raises(KeyError):
        eng.fork("nobody")


def test_fork_keeps_log_probabilities():
    """A fork's log-probabilities are its outputs', one by one, those it keeps among them; one that asks for what
    the request does not have is refused."""
    prompt = [3, 1, 4, 1, 5, 9, 2, 6]
    eng = _engine()
    rid = eng.add_request(prompt, SamplingParams(max_tokens=12, logprobs=2))
    plain = eng.add_request(prompt, SamplingParams(max_tokens=12))
    for _ in range(6):
        eng.step()
    twin, back = eng.fork(rid), eng.fork(rid, SamplingParams(max_tokens=12, logprobs=1), keep=11)
    for args in ((plain, SamplingParams(max_tokens=12, logprobs=1)), (rid, SamplingParams(max_tokens=12, logprobs=3))):
        with pytest.raises(ValueError):
            eng.fork(*args)
    while eng.has_work():
        eng.step()
    want = eng.request(rid)
    assert len(want.logprobs) == 12
    for other, k in ((twin, 2), (back, 1)):
        req = eng.request(other)
        assert req.outputs == want.outputs and len(req.logprobs) == 12
        for (lp, top), (wlp, wtop) in zip(req.logprobs, want.logprobs):
            assert abs(lp - wlp) < 1e-4 and [t for t, _ in top] == [t for t, _ in wtop[:k]]
    silent = _engine()
    rid = silent.add_request(prompt, SamplingParams(max_tokens=6, logprobs=2))
    silent.step()
    none = silent.fork(rid, SamplingParams(max_tokens=6))
    while silent.has_work():
        silent.step()
    assert silent.request(none).logprobs == [] and silent.request(none).outputs == silent.request(rid).outputs


def test_fork_of_outputs_that_end_it_is_refused():
    """Kept outputs that reach the fork's max_tokens, or end with one of its stop ids, leave nothing to continue."""
    eng = _engine()
    rid = eng.add_request([3, 1, 4, 1, 5, 9, 2, 6], SamplingParams(max_tokens=12))
    for _ in range(5):
        eng.step()
    eng.flush()
    out = list(eng.request(rid).outputs)
    last = dict(max_tokens=12, stop_ids=(out[-1],))
    for params in (SamplingParams(max_tokens=len(out)), SamplingParams(max_tokens=2), SamplingParams(**last),
                   SamplingParams(max_tokens=12, eos_id=out[-1], ignore_eos=False)):
        with pytest.raises(ValueError):
            eng.fork(rid, params)
    assert len(eng.scheduler.running) == 1 and eng.blocks.shared_blocks == 0
    one = eng.fork(rid, SamplingParams(max_tokens=len(out) + 1))
    two = eng.fork(rid, SamplingParams(max_tokens=2), keep=9)
    while eng.has_work():
        eng.step()
    want = eng.request(rid).outputs
    assert eng.request(one).outputs == want[: len(out) + 1] and eng.request(two).outputs == want[:2]


def test_fork_limits_and_preemption():
    eng = _engine(max_batch=2, num_blocks=8)
    rid = eng.add_request(list(range(1, 40)), SamplingParams(max_tokens=40))
    eng.step()
    for keep in (0, 41):
        with pytest.raises(ValueError):
            eng.fork(rid, keep=keep)
    twin = eng.fork(rid)
    with pytest.raises(RuntimeError):
        eng.fork(rid)
    want = _engine().generate([list(range(1, 40))], max_tokens=40)[0]
    while eng.has_work():  # 8 blocks do not hold both to the end: one is preempted and recomputed
        eng.step()
    assert eng.request(rid).outputs == want and eng.request(twin).outputs == want
    assert eng.blocks.free_blocks == 8
    tight = _engine(num_blocks=3)
    rid = tight.add_request(list(range(1, 40)), SamplingParams(max_tokens=2))
    tight.step()
    with pytest.raises(MemoryError):
        tight.fork(rid)


def test_prefill_step_carries_its_lengths():
    eng = _engine(kv_quant="int4")
    for n in (19, 3):
        eng.add_request(list(range(1, n + 1)), SamplingParams(max_tokens=4))
    inp = eng.executor.worker.runner.prefill_input(eng.scheduler.schedule())
    assert inp.lengths == [(19, 19), (3, 3)] and inp.max_context == 19

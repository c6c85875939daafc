"""Scoring and log-probability requests that fail, or that must not be taken, through the engine (CPU)."""

import pytest
import torch

from b200serve.core.config import EngineConfig
from b200serve.engine.b200_engine import B200Engine
from b200serve.engine.sampler import SamplingParams
from b200serve.models.config import BUILTIN
from b200serve.models.weights import random_weights


@pytest.fixture(scope="module")
def engine():
    w = random_weights(BUILTIN["tiny-qwen2"], seed=0, dtype=torch.float32)
    eng = B200Engine(EngineConfig(model="tiny-qwen2", device="cpu", dtype="float32", cuda_graphs=False, max_seq=128,
                                  max_batch=4), weights=w)
    eng.load()
    yield eng
    eng.unload()


def test_a_failed_score_raises(engine, monkeypatch):
    """A runner whose score raises fails the caller, whichever of its prompts that was."""
    real = engine.runner.score

    def score(hidden, tokens):
        if 99 in tokens.tolist():
            raise MemoryError("no room for the partial results")
        return real(hidden, tokens)

    monkeypatch.setattr(engine.runner, "score", score)
    for prompts in ([[1, 2, 99, 4]], [[1, 2, 3], [4, 5, 6, 7], [8, 99]]):
        with pytest.raises(RuntimeError, match="scoring failed"):
            engine.score(prompts, timeout=60)
    monkeypatch.undo()
    [ok] = engine.score([[1, 2, 3, 4]], timeout=60)          # the engine goes on
    assert len(ok["logprobs"]) == len(ok["entropy"]) == 3


def test_a_refused_prompt_queues_nothing(engine):
    seen = []
    real = engine.scheduler.add_embedding
    engine.scheduler.add_embedding = lambda r: (seen.append(r), real(r))[1]
    try:
        for bad in ([1] * 128, [], [32000], [-1]):
            with pytest.raises(ValueError):
                engine.score([[1, 2, 3], bad], timeout=60)
    finally:
        del engine.scheduler.add_embedding
    assert not seen and not engine.scheduler.embed_waiting


def test_a_prompt_larger_than_the_cache_is_refused():
    w = random_weights(BUILTIN["tiny-qwen2"], seed=0, dtype=torch.float32)
    eng = B200Engine(EngineConfig(model="tiny-qwen2", device="cpu", dtype="float32", cuda_graphs=False, max_seq=128,
                                  max_batch=1, kv_blocks=4), weights=w)
    try:
        with pytest.raises(ValueError, match="KV cache"):
            eng.score([[1] * 65], timeout=3)
        [ok] = eng.score([[1] * 64], timeout=60)
        assert len(ok["logprobs"]) == 63
    finally:
        eng.unload()


def test_a_failed_score_leaves_other_requests_alone(engine, monkeypatch):
    """A generation under way, and another scoring call of the same step, end as they would without it."""
    def score(hidden, tokens):
        if 99 in tokens.tolist():
            raise MemoryError("no room for the partial results")
        return real(hidden, tokens)

    from b200serve.engine.scheduler import Request
    real = engine.runner.score
    prompt, params = list(range(10, 30)), SamplingParams(max_tokens=40, ignore_eos=True)
    [want] = engine.generate([prompt], params, timeout=60)
    monkeypatch.setattr(engine.runner, "score", score)
    req = engine.submit(Request(prompt=prompt, params=params))
    good = engine.scheduler.add_scoring(Request(prompt=[5, 6, 7], params=SamplingParams(max_tokens=1)))
    with pytest.raises(RuntimeError, match="no room"):
        engine.score([[1, 99]], timeout=60)
    assert req.done_event.wait(60) and good.done_event.wait(60)
    assert req.finish_reason == "length" and req.output == want.output and len(good.scores[0]) == 2


def test_logprobs_switch_takes_truth_values():
    for value, n in ((False, -1), (None, -1), (True, 0), (0, 0), (7, 7), (-1, -1)):
        assert SamplingParams.from_dict({"logprobs": value}).logprobs == n
        assert SamplingParams(logprobs=value).logprobs == n
        assert type(SamplingParams(logprobs=value).logprobs) is int
    assert SamplingParams.from_dict({}).logprobs == SamplingParams().logprobs == -1


def test_streaming_ignores_logprobs(engine, monkeypatch):
    """A text stream returns no records, so the key neither slows its requests nor refuses them."""
    seen = []
    real = engine.submit
    monkeypatch.setattr(engine, "submit", lambda r: (seen.append(r), real(r))[1])
    msgs = [{"role": "user", "content": "hi"}]
    want = engine.generate_streaming(msgs, 4, 0.0, sampling={"top_k": 1})
    for value in (5, 50, True, False, "many"):
        assert engine.generate_streaming(msgs, 4, 0.0, sampling={"top_k": 1, "logprobs": value}) == want
    assert len(seen) == 6 and all(r.params.logprobs == -1 and r.logprobs == [] for r in seen)


def test_a_wait_that_ran_out_fails_the_score(engine, monkeypatch):
    from b200serve import ops
    codes = [13]
    monkeypatch.setattr(ops, "linear_logprobs_error", lambda reset=True: codes.pop() if codes else 0)
    with pytest.raises(RuntimeError, match="code 13"):
        engine.score([[1, 2, 3]], timeout=60)
    [ok] = engine.score([[1, 2, 3]], timeout=60)
    assert len(ok["logprobs"]) == 2


def test_pages_of_a_failed_step_stay_out_of_the_prefix_cache(engine, monkeypatch):
    """A step that ends in an exception after its forward may have written anything into its pages."""
    prompt, params = list(range(200, 260)), SamplingParams(max_tokens=4, ignore_eos=True)

    def failing(logits, reqs):
        raise RuntimeError("the step's results are void")

    monkeypatch.setattr(engine.scheduler, "_sample", failing)
    [req] = engine.generate([prompt], params, timeout=60)
    assert req.finish_reason == "error"
    monkeypatch.undo()
    [again] = engine.generate([prompt], params, timeout=60)
    assert again.finish_reason == "length" and again.prefix_hit == 0
    [third] = engine.generate([prompt], params, timeout=60)
    assert third.prefix_hit > 0 and third.output == again.output


def test_a_layer_that_gave_up_fails_its_step(engine, monkeypatch):
    """The error word of the fused MoE layer is looked at before a step's tokens, embeddings or scores are taken."""
    from b200serve import ops
    codes, asked = [], []

    def error(reset=True, wait=True):
        asked.append(wait)
        return codes.pop() if codes else 0

    monkeypatch.setattr(ops, "moe_layer_error", error)
    prompt = list(range(300, 330))
    for params in (SamplingParams(max_tokens=4, ignore_eos=True), SamplingParams(max_tokens=4, logprobs=2)):
        codes.append(24)
        [req] = engine.generate([prompt], params, timeout=60)
        assert req.finish_reason == "error" and req.output == []
        [req] = engine.generate([prompt], params, timeout=60)
        assert req.finish_reason in ("length", "stop") and req.prefix_hit in (0, 16)
    codes.append(24)
    with pytest.raises(RuntimeError, match="code 24"):
        engine.score([[1, 2, 3]], timeout=60)
    codes.append(24)
    with pytest.raises(RuntimeError, match="embedding failed"):
        engine.embed(["a few words"], timeout=60)
    assert asked and not any(asked)                          # never waits for the GPU


def test_a_worker_rank_stops_after_a_layer_gave_up(monkeypatch):
    from types import SimpleNamespace

    from b200serve import ops
    from b200serve.parallel import worker
    monkeypatch.setattr(ops, "moe_layer_error", lambda reset=True, wait=True: 24)
    comm = SimpleNamespace(broadcast=lambda t, src: t.copy_(torch.tensor([worker.OP_PIPE_STEP] + [0] * (len(t) - 1))))
    runner = SimpleNamespace(device="cpu", pipeline_step=lambda slot: None)
    with pytest.raises(RuntimeError, match="code 24"):
        worker.worker_loop(runner, comm)


def _with_generation(engine, start):
    """``start()`` while a generation is under way, which has to end as it would alone; what start() raised or returned."""
    from b200serve.engine.scheduler import Request
    prompt, params = list(range(10, 30)), SamplingParams(max_tokens=40, ignore_eos=True)
    [want] = engine.generate([prompt], params, timeout=60)
    req = engine.submit(Request(prompt=prompt, params=params))
    try:
        out = start()
    except RuntimeError as e:
        out = e
    assert req.done_event.wait(60) and req.finish_reason == "length" and req.output == want.output
    return out


def test_a_failed_embedding_step_leaves_generations_alone(engine, monkeypatch):
    real = engine.runner.prefill

    def prefill(seqs):
        if any(s.get("hidden") for s in seqs):
            raise MemoryError("no room for the activations")
        return real(seqs)

    monkeypatch.setattr(engine.runner, "prefill", prefill)
    free = engine.scheduler.alloc.num_free
    for call in (lambda: engine.score([[1, 2, 3], [4, 5]], timeout=60), lambda: engine.embed(["some text"], timeout=60)):
        out = _with_generation(engine, call)
        assert isinstance(out, RuntimeError) and "no room for the activations" in str(out)
    monkeypatch.undo()
    assert engine.scheduler.alloc.num_free == free and len(engine.score([[1, 2, 3]], timeout=60)[0]["logprobs"]) == 2


def test_a_void_step_fails_all_of_its_inputs(engine, monkeypatch):
    """One prefill, one error word: the first input that reads it must not clear it for the others."""
    from b200serve import ops
    from b200serve.engine.scheduler import Request
    codes = []
    monkeypatch.setattr(ops, "moe_layer_error", lambda reset=True, wait=True: codes.pop() if codes else 0)
    params = SamplingParams(max_tokens=1)
    reqs = [Request(prompt=p, params=params) for p in ([1, 2, 3], [4, 5, 6], [7, 8])]
    engine.stop_loop()                                       # the three of them in one step
    for r in reqs[:2]:
        engine.scheduler.add_scoring(r)
    engine.scheduler.add_embedding(reqs[2])
    codes.append(24)
    engine.scheduler._embed_step()
    assert all(r.done_event.is_set() and "code 24" in str(r.error) and r.finish_reason == "error" for r in reqs)
    assert all(r.scores is None and r.embedding is None for r in reqs)


def test_a_call_that_timed_out_leaves_nothing_queued(engine, monkeypatch):
    monkeypatch.setattr(engine.scheduler, "step", lambda: 0)             # a step that takes for ever
    monkeypatch.setattr(engine.scheduler, "has_work", lambda: False)
    with pytest.raises(TimeoutError):
        engine.score([[1, 2, 3], [4, 5, 6]], timeout=0.2)
    assert engine.scheduler.embed_waiting == []
    monkeypatch.undo()
    assert len(engine.score([[1, 2, 3]], timeout=60)[0]["logprobs"]) == 2

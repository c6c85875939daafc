"""Log probabilities through the engine (CPU): sampled tokens with alternatives, and scoring of given tokens."""

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
    yield eng
    eng.unload()


def _prompt(n, seed=0):
    return torch.randint(0, 32000, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _rows(eng, tokens):
    """Log probabilities of every next token of ``tokens``, from the logits of one prefill."""
    eng.load()
    bt = eng.scheduler.alloc.allocate((len(tokens) + 15) // 16)
    try:
        logits = eng.runner.prefill([{"ids": tokens, "start": 0, "block_table": bt, "all_logits": True}])
    finally:
        eng.scheduler.alloc.release(bt)
    return torch.log_softmax(logits.double(), -1)


def test_score_matches_the_logits(engine):
    prompts = [_prompt(40), _prompt(7, 1), _prompt(1, 2)]
    got = engine.score(prompts)
    for p, r in zip(prompts, got):
        assert r["tokens"] == p and len(r["logprobs"]) == len(r["entropy"]) == len(p) - 1
        if len(p) > 1:
            lp = _rows(engine, p)[:-1]
            want = lp.gather(1, torch.tensor(p[1:])[:, None])[:, 0]
            assert torch.allclose(torch.tensor(r["logprobs"]).double(), want, atol=1e-4)
            assert torch.allclose(torch.tensor(r["entropy"]).double(), -(lp.exp() * lp).sum(-1), atol=1e-3)


def test_score_refuses(engine):
    with pytest.raises(ValueError):
        engine.score([[]])
    with pytest.raises(ValueError):
        engine.score([[32000]])
    with pytest.raises(ValueError):
        engine.score([[-1]])
    with pytest.raises(ValueError):
        engine.score([_prompt(128)])


@pytest.mark.parametrize("params", [dict(temperature=0.0), dict(temperature=0.8, seed=3),
                                    dict(temperature=0.0, repeat_penalty=1.5, presence_penalty=2.0)])
def test_sampled_tokens_report_log_probabilities(engine, params):
    prompt = _prompt(20)
    sp = SamplingParams(max_tokens=6, ignore_eos=True, **params)
    [plain] = engine.generate([prompt], sp)
    [req] = engine.generate([prompt], SamplingParams(max_tokens=6, ignore_eos=True, logprobs=4, **params))
    assert req.output == plain.output and plain.logprobs == []
    assert [e["token"] for e in req.logprobs] == req.output
    lp = _rows(engine, prompt + req.output)[len(prompt) - 1:-1]
    for row, e in zip(lp, req.logprobs):
        assert abs(e["logprob"] - float(row[e["token"]])) < 1e-4      # before penalties and temperature
        assert e["rank"] == int((row > row[e["token"]]).sum())
        assert [t for t, _ in e["top"]] == row.topk(4).indices.tolist()


def test_logprobs_mixes_with_other_requests_and_is_bounded(engine):
    a, b = _prompt(9, 4), _prompt(12, 5)
    eng_reqs = [engine.submit(r) for r in _requests([(a, 2), (b, -1)])]
    for r in eng_reqs:
        assert r.done_event.wait(60)
    assert len(eng_reqs[0].logprobs) == 4 and eng_reqs[1].logprobs == []
    with pytest.raises(ValueError):
        engine.generate([a], SamplingParams(max_tokens=1, logprobs=33))


def _requests(specs):
    from b200serve.engine.scheduler import Request
    return [Request(prompt=p, params=SamplingParams(max_tokens=4, ignore_eos=True, logprobs=n)) for p, n in specs]

"""Log probabilities and the fused MoE layer through the engine on the GPU."""

import pytest
import torch

from b200serve import ops
from b200serve.core.config import EngineConfig
from b200serve.engine.b200_engine import B200Engine
from b200serve.engine.sampler import SamplingParams

pytestmark = pytest.mark.gpu


def _engine(model, **kw):
    return B200Engine(EngineConfig(model=model, max_batch=4, max_seq=256, kv_blocks=64, **kw))


def _prompt(n, seed=0):
    return torch.randint(0, 32000, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _rows(eng, tokens):
    bt = eng.scheduler.alloc.allocate((len(tokens) + 15) // 16)
    try:
        return eng.runner.prefill([{"ids": tokens, "start": 0, "block_table": bt, "all_logits": True}])
    finally:
        eng.scheduler.alloc.release(bt)


@pytest.mark.parametrize("graphs", [True, False])
def test_generate_and_score(graphs):
    eng = _engine("tiny-qwen2", cuda_graphs=graphs)
    try:
        prompt = _prompt(50)
        [plain] = eng.generate([prompt], SamplingParams(max_tokens=12, ignore_eos=True), timeout=300)
        [req] = eng.generate([prompt], SamplingParams(max_tokens=12, ignore_eos=True, logprobs=5), timeout=300)
        assert req.output == plain.output and len(req.logprobs) == 12
        for e in req.logprobs:                                # greedy: the token leads its alternatives
            assert e["rank"] == 0 and e["top"][0][0] == e["token"] and e["top"][0][1] == e["logprob"]
            assert [p for _, p in e["top"]] == sorted((p for _, p in e["top"]), reverse=True)
        [sc] = eng.score([prompt])
        logits = _rows(eng, prompt)[:-1]
        ref = ops.token_logprobs(logits, torch.tensor(prompt[1:], device=logits.device))
        # the same bf16 hidden states; the head's sums only differ in their order
        assert torch.allclose(torch.tensor(sc["logprobs"]), ref.logprob.cpu(), atol=1e-4)
        assert torch.allclose(torch.tensor(sc["entropy"]), ref.entropy.cpu(), atol=1e-3)
        assert ops.linear_logprobs_error() == 0
    finally:
        eng.unload()


def test_penalties_do_not_enter_the_log_probabilities():
    eng = _engine("tiny-qwen2")
    try:
        prompt = _prompt(30, 3)
        kw = dict(max_tokens=6, ignore_eos=True, repeat_penalty=1.8, presence_penalty=1.0, frequency_penalty=0.5)
        [req] = eng.generate([prompt], SamplingParams(logprobs=0, **kw), timeout=300)
        logits = _rows(eng, prompt + req.output)[len(prompt) - 1:-1]
        ref = ops.token_logprobs(logits, torch.tensor(req.output, device=logits.device))
        # decode and prefill differ by bf16 roundings of the hidden state (2^-8 of each element, logits of std 0.3)
        assert torch.allclose(torch.tensor([e["logprob"] for e in req.logprobs]), ref.logprob.cpu(), atol=0.05)
    finally:
        eng.unload()


def test_fused_moe_layers_in_the_engine():
    prompt = _prompt(40, 1)
    logits = {}
    for fused in (False, True):
        eng = _engine("tiny-qwen3-moe", moe_fused=fused)
        try:
            eng.load()
            calls = []
            real = ops.moe_layer
            ops.moe_layer = lambda *a, **k: (calls.append(1), real(*a, **k))[1]
            try:
                [req] = eng.generate([prompt], SamplingParams(max_tokens=8, ignore_eos=True, logprobs=3), timeout=300)
            finally:
                ops.moe_layer = real
            assert len(req.output) == 8 and bool(calls) == fused
            bt = eng.scheduler.alloc.allocate(3)
            eng.runner.prefill([{"ids": prompt, "start": 0, "block_table": bt}])
            out, _ = eng.runner.decode([5], [len(prompt)], [bt[len(prompt) // 16] * 16 + len(prompt) % 16], [bt],
                                       [len(prompt) + 1], greedy=False)
            logits[fused] = out.float().cpu().clone()
        finally:
            eng.unload()
    assert ops.moe_layer_error() == 0
    d = (logits[True] - logits[False]).norm() / logits[False].norm()
    # two layers whose outputs are rounded to bf16 at other places: a few 2^-8 of the norm
    assert float(d) < 4 * 2.0 ** -8

"""Scoring through the engine with capped logits and with a quantised LM head, several prompts to a step, and the fused
MoE layer on a rank that holds a share of the experts."""

from types import SimpleNamespace

import pytest
import torch

from b200serve import ops
from b200serve.core.config import EngineConfig
from b200serve.engine.b200_engine import B200Engine
from b200serve.engine.sampler import SamplingParams
from b200serve.models.config import BUILTIN, ModelConfig
from b200serve.models.moe import MoEBlock

pytestmark = pytest.mark.gpu


def _prompt(n, seed=0):
    return torch.randint(0, 32000, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _reference(eng, tokens):
    """(log probabilities, entropies) of tokens[1:] from the logits of one prefill."""
    bt = eng.scheduler.alloc.allocate((len(tokens) + 15) // 16)
    try:
        logits = eng.runner.prefill([{"ids": tokens, "start": 0, "block_table": bt, "all_logits": True}])
    finally:
        eng.scheduler.alloc.release(bt)
    logp = torch.log_softmax(logits[:-1].double().cpu(), -1)
    return logp.gather(1, torch.tensor(tokens[1:])[:, None])[:, 0], -(logp.exp() * logp).sum(-1)


@pytest.mark.parametrize("cap", [0.5, 30.0])
def test_capped_logits(cap):
    """Prompts of 40 and 150 tokens: one and two CTAs per tile, against 64 bits from the hidden states that the step had
    (how the prompts share steps is open, and moves them by bf16 roundings). A logit differs by 256 fp32
    additions at most (256 * 2^-24 of logits below 4) and by the tanh (2^-21 cap)."""
    cfg = ModelConfig("tiny-cap", 32000, 256, 2, 4, 2, 64, 688, attn_bias=True, final_softcap=cap)
    eng = B200Engine(EngineConfig(model="tiny-cap", max_batch=4, max_seq=256, kv_blocks=64, init_std=0.1), model_config=cfg)
    try:
        eng.load()
        prompts, seen, real = [_prompt(40), _prompt(150, 1)], {}, eng.runner.score

        def score(hidden, tokens):
            seen[tuple(tokens.tolist())] = hidden.clone()
            return real(hidden, tokens)

        eng.runner.score = score
        got = eng.score(prompts)
        w = eng.weights.lm_head.unpacked().double().cpu()
        for p, r in zip(prompts, got):
            z = seen[tuple(p[1:])].double().cpu() @ w.t()
            logp = torch.log_softmax(cap * torch.tanh(z / cap), -1)
            lp, ent = logp.gather(1, torch.tensor(p[1:])[:, None])[:, 0], -(logp.exp() * logp).sum(-1)
            err = 256 * 2.0 ** -24 * 4 + 2 * cap * 2.0 ** -21
            tol = 2 * err + 1e-5                        # and the statistics' own 1e-5 (32000 terms)
            assert float((torch.tensor(r["logprobs"]).double() - lp).abs().max()) < tol
            assert float((torch.tensor(r["entropy"]).double() - ent).abs().max()) < 21 * err + 2e-4   # 2 ln V = 21
        assert ops.linear_logprobs_error() == 0
    finally:
        eng.unload()


def test_quantised_head():
    """More than one pass of 512 rows. A path may round its dequantised weights to bf16 (2^-8 each): a logit of root mean
    square 0.3 moves by 2^-8 of that, five times as much for the largest of 22 M, on either side."""
    cfg = ModelConfig("tiny-q", 32000, 256, 2, 4, 2, 64, 512, attn_bias=True)
    eng = B200Engine(EngineConfig(model="tiny-q", max_batch=2, max_seq=1024, kv_blocks=80, quantize="q4_k_m"),
                     model_config=cfg)
    try:
        eng.load()
        assert isinstance(eng.weights.lm_head, ops.QuantWeight)
        tokens = _prompt(700, 2)
        [r] = eng.score([tokens])
        lp, ent = _reference(eng, tokens)
        tol = 2 * 5 * 2.0 ** -8 * 0.3
        assert len(r["logprobs"]) == 699
        assert float((torch.tensor(r["logprobs"]).double() - lp).abs().max()) < tol
        assert float((torch.tensor(r["entropy"]).double() - ent).abs().max()) < tol
        [req] = eng.generate([tokens[:50]], SamplingParams(max_tokens=5, ignore_eos=True, logprobs=0), timeout=300)
        assert len(req.logprobs) == 5 and all(e["rank"] == 0 and e["top"] == [] for e in req.logprobs)
    finally:
        eng.unload()


def _blocks(cfg, ranks):
    """The fused MoE blocks of ``ranks`` expert-parallel ranks with the same weights, one after another."""
    g = torch.Generator(device="cuda").manual_seed(0)
    E, H, I = cfg.num_experts, cfg.hidden_size, cfg.moe_intermediate_size
    rnd = lambda *s, f=1.0: (torch.randn(*s, device="cuda", generator=g) * f).bfloat16()
    router, gu, dn = rnd(E, H, f=1.4 / H ** 0.5), rnd(E, 2 * I, H, f=H ** -0.5), rnd(E, H, I, f=I ** -0.5)
    for r in range(ranks):
        sl = slice(r * E // ranks, (r + 1) * E // ranks)
        lw = SimpleNamespace(router=ops.pack_weight(router), experts_gate_up=gu[sl], experts_down=dn[sl],
                             shared_gate_up=None)
        b = MoEBlock(cfg, SimpleNamespace(layers=[lw], ep_size=ranks, ep_rank=r), device="cuda")
        assert b.use_fused()
        yield b


@pytest.mark.parametrize("T", [1, 5, 16])
@pytest.mark.parametrize("ranks", [2, 4])
def test_the_ranks_shares_add_up(T, ranks):
    cfg = BUILTIN["tiny-qwen3-moe"]
    x = torch.randn(T, cfg.hidden_size, device="cuda", generator=torch.Generator(device="cuda").manual_seed(T)).bfloat16()
    [whole] = [b(0, x).float() for b in _blocks(cfg, 1)]
    shares = [b(0, x).float() for b in _blocks(cfg, ranks)]
    # every output is rounded once (2^-8 of itself); the sums' own errors are far below 2^-12 of the terms
    bound = 2.0 ** -8 * (whole.abs() + sum(s.abs() for s in shares)) + 2.0 ** -12 * whole.abs().max()
    assert bool(((sum(shares) - whole).abs() <= bound).all())
    assert ops.moe_layer_error() == 0


def test_a_model_sized_layer():
    """128 experts of 768 over 2048, 8 per token: 1, 4, 8 and 16 rows against the 64-bit reference."""
    from logprob_cases import MoECase
    c = MoECase(T=16, H=2048, E=128, k=8, inner=768)
    a = list(c.args("cuda"))
    ref, bound = c.reference()
    for T in (1, 4, 8, 16):
        out = ops.moe_layer(a[0][:T], *a[1:])
        assert bool(((out.double().cpu() - ref[:T]).abs() <= bound[:T]).all())
        # rounding to bf16 leaves at most 2^-8, 2^-9 / sqrt 3 * 2 = 0.0023 on average, and the rest adds nothing to it
        rel = (out.double().cpu() - ref[:T]).norm() / ref[:T].norm()
        assert float(rel) < 2.0 ** -8 / 3 ** 0.5 + 1e-4
    assert ops.moe_layer_error() == 0

"""The small-batch MoE layer against a 64-bit reference: odd sizes, experts of other ranks, strided rows, equal
router logits, repeats, streams and graphs."""

import pytest
import torch

from b200serve import ops
from logprob_cases import NAN, MoECase

pytestmark = pytest.mark.gpu
dev = "cuda"


@pytest.fixture(autouse=True)
def _ext():
    ops.ext()


def _check(c, out, rows=None):
    ref, bound = c.reference()
    d = (out.double().cpu() - ref).abs()
    assert bool((d <= bound).all()), float((d - bound).max())
    assert ops.moe_layer_error() == 0


@pytest.mark.parametrize("case", [
    dict(T=1, H=8, E=1, k=1, inner=1), dict(T=1, H=64, E=4, k=2, inner=64), dict(T=2, H=256, E=16, k=4, inner=128),
    dict(T=5, H=200, E=9, k=3, inner=70), dict(T=8, H=1000, E=33, k=5, inner=300), dict(T=9, H=136, E=7, k=7, inner=257),
    dict(T=16, H=512, E=64, k=8, inner=192), dict(T=16, H=264, E=2, k=1, inner=520), dict(T=3, H=2048, E=8, k=2, inner=1400),
    dict(T=16, H=128, E=256, k=16, inner=64), dict(T=4, H=4096, E=4, k=2, inner=65, renorm=False),
    dict(T=7, H=128, E=16, k=4, inner=96, first=8, local=8), dict(T=16, H=128, E=16, k=2, inner=96, first=15, local=1)],
    ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()))
def test_moe_layer(case):
    c = MoECase(**case)
    a = c.args(dev)
    out = ops.moe_layer(*a)
    assert out.dtype == torch.bfloat16 and out.shape == (c.T, c.H)
    _check(c, out)
    for _ in range(3):                      # the order in which CTAs take units does not show
        assert torch.equal(ops.moe_layer(*a), out)


def test_no_row_has_an_expert_here():
    c = MoECase(T=6, H=192, E=12, k=2, inner=128, first=0, local=3)
    a = list(c.args(dev))
    z = torch.zeros(12, 192)
    z[:, 0] = torch.arange(12.0)            # experts 10 and 11 for every row with x[0] > 0
    a[1] = z.bfloat16().to(dev)
    a[0][:, 0] = 1.0
    out = ops.moe_layer(*a)
    assert bool((out == 0).all()) and ops.moe_layer_error() == 0


def test_equal_router_logits_take_the_lowest_ids():
    c = MoECase(T=3, H=128, E=40, k=4, inner=64)
    c.router.zero_()
    _check(c, ops.moe_layer(*c.args(dev)))


def test_all_rows_on_the_same_experts_and_out_rows():
    c = MoECase(T=16, H=320, E=8, k=2, inner=128)
    c.x[:] = c.x[0]
    wide = torch.full((16, 384), 7.0, dtype=torch.bfloat16, device=dev)
    a = list(c.args(dev))
    src = torch.zeros(16, 384, dtype=torch.bfloat16, device=dev)
    src[:, 8:328] = a[0]
    a[0] = src[:, 8:328]                    # strided rows in and out
    out = ops.moe_layer(*a, out=wide[:, 16:336])
    _check(c, out)
    assert bool((wide[:, :16] == 7).all() and (wide[:, 336:] == 7).all())
    assert bool((out == out[0]).all())


def test_a_bad_row_stays_alone():
    c = MoECase(T=12, H=256, E=16, k=2, inner=128)
    a = list(c.args(dev))
    good = ops.moe_layer(*a)
    a[0] = a[0].clone()
    a[0][4, 9] = NAN
    got = ops.moe_layer(*a)
    keep = torch.arange(12, device=dev) != 4
    assert torch.equal(got[keep], good[keep]) and bool(got[4].isnan().all())


def test_streams_and_graphs():
    c1, c2 = MoECase(T=4, H=512, E=32, k=4, inner=256, seed=1), MoECase(T=16, H=512, E=32, k=4, inner=256, seed=2)
    a1, a2 = c1.args(dev), c2.args(dev)
    w1, w2 = ops.moe_layer(*a1), ops.moe_layer(*a2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(8):                      # two calls at once
        with torch.cuda.stream(side):
            outs.append((ops.moe_layer(*a2), w2))
        outs.append((ops.moe_layer(*a1), w1))
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        outs.append((ops.moe_layer(*a1), w1))
    with torch.cuda.graph(g2):
        outs.append((ops.moe_layer(*a2), w2))
    for _ in range(3):
        g1.replay()
        g2.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in outs) and ops.moe_layer_error() == 0


def test_decode_tail_moe_norm_scoring():
    """One decode step's tail as it is used: MoE layer -> add + RMSNorm -> LM head scoring, against 64 bits."""
    c = MoECase(T=6, H=256, E=16, k=4, inner=128)
    a = c.args(dev)
    g = torch.Generator().manual_seed(5)
    w_norm = (1 + 0.1 * torch.randn(256, generator=g)).bfloat16()
    head = (torch.randn(4001, 256, generator=g) * 0.1).bfloat16()
    tokens = torch.randint(0, 4001, (6,), generator=g)
    y = ops.moe_layer(*a)
    h = ops.rmsnorm(y, w_norm.to(dev), 1e-6, residual=a[0])
    lp, ent = ops.linear_logprobs(h, ops.PackedWeight(head.to(dev)), tokens.to(dev))
    ref, _ = c.reference()
    s = ref + c.x.double()
    n = s * torch.rsqrt(s.pow(2).mean(-1, keepdim=True) + 1e-6) * w_norm.double()
    logp = torch.log_softmax(n @ head.double().t(), -1)
    # bf16 roundings on the way (the layer's output, the sum, the norm, its product): four of at most 2^-8 of
    # each element of h; a logit moves by at most 4 * 2^-8 |h| |w|, by its root-sum-square in practice
    bound = 2 * 4 * 2.0 ** -8 * float((n.abs() @ head.double().abs().t()).max())
    assert float((lp.double().cpu() - logp.gather(1, tokens[:, None])[:, 0]).abs().max()) < bound
    assert float((ent.double().cpu() + (logp.exp() * logp).sum(-1)).abs().max()) < bound * 2 * 8.3
    logits = ops.linear(h, ops.PackedWeight(head.to(dev)), epilogue=ops.EPI_F32)
    two = ops.token_logprobs(logits, tokens.to(dev), top=3)
    assert float((two.logprob - lp).abs().max()) < 1e-4


def test_refusals_on_the_gpu():
    c = MoECase(T=2, H=64, E=4, k=2, inner=64)
    a = list(c.args(dev))

    def but(i, v):
        b = list(a)
        b[i] = v
        return b

    odd = torch.zeros(3, 70, device=dev).bfloat16()
    for bad in (but(0, a[0].float()), but(0, odd[:2, 1:65]), but(0, torch.zeros(17, 64, device=dev).bfloat16()),
                but(1, a[1].float()), but(1, a[1].cpu()), but(2, a[2].cpu()), but(2, a[2][:-64]), but(3, 96), but(4, a[4][:-1]),
                but(5, 128), but(6, 0), but(6, 5), but(8, 1), but(8, -1)):
        with pytest.raises((RuntimeError, ValueError)):
            ops.moe_layer(*bad)
    with pytest.raises(RuntimeError):
        ops.moe_layer(*a, out=torch.empty(2, 64, device=dev))

"""Log-probability operators and the small-batch MoE layer on the CPU path, against 64-bit references,
and what they refuse."""

import pytest
import torch

from b200serve import ops
from logprob_cases import INF, NAN, MoECase, check_linear_logprobs, check_token_logprobs


def test_token_logprobs_ties_masks_and_bad_rows():
    x = torch.full((7, 9), -INF)
    x[0] = torch.tensor([1.0, 3.0, 3.0, 2.0, -1.0, 3.0, 0.0, -0.0, 0.5])
    x[1, 4] = 2.0                                  # one entry left
    x[3] = torch.arange(9.0)
    x[3, 2] = NAN
    x[4] = torch.arange(9.0)
    x[4, 0] = INF
    x[5] = 0.0
    x[6] = torch.randn(9)
    tokens = torch.tensor([7, 4, 3, 1, 1, 8, 9])   # row 6: no such token
    check_token_logprobs(ops.token_logprobs(x, tokens, top=5), x, tokens, 5)
    check_token_logprobs(ops.token_logprobs(x, tokens.int(), top=12), x, tokens, 12)
    check_token_logprobs(ops.token_logprobs(x, tokens), x, tokens, 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_logprobs_random(dtype):
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(5, 1003, generator=g) * 3).to(dtype)
    tokens = torch.randint(0, 1003, (5,), generator=g)
    check_token_logprobs(ops.token_logprobs(x, tokens, top=20), x, tokens, 20)
    wide = torch.empty(5, 1100, dtype=dtype)
    wide[:, :1003] = x                             # strided rows
    check_token_logprobs(ops.token_logprobs(wide[:, :1003], tokens, top=4), x, tokens, 4)


@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_linear_logprobs_is_token_logprobs_of_the_product(softcap):
    g = torch.Generator().manual_seed(4)
    x, w = torch.randn(6, 72, generator=g).bfloat16(), (torch.randn(301, 72, generator=g) * 0.2).bfloat16()
    tokens = torch.tensor([0, 300, 17, -1, 301, 5])
    got = ops.linear_logprobs(x, w, tokens, softcap=softcap)
    check_linear_logprobs(got, x, w, tokens, softcap)
    packed = ops.linear_logprobs(x, ops.PackedWeight(w), tokens, softcap=softcap)
    assert all(torch.equal(a, b) or torch.allclose(a, b, equal_nan=True) for a, b in zip(got, packed))


@pytest.mark.parametrize("case", [dict(T=1, H=64, E=4, k=2, inner=64), dict(T=5, H=200, E=9, k=3, inner=70),
                                  dict(T=4, H=64, E=8, k=2, inner=33, first=4, local=4, renorm=False),
                                  dict(T=16, H=128, E=5, k=5, inner=100), dict(T=0, H=64, E=4, k=2, inner=64)])
def test_moe_layer_cpu(case):
    c = MoECase(**case)
    out = ops.moe_layer(*c.args())
    ref, bound = c.reference()
    assert out.dtype == torch.bfloat16 and out.shape == c.x.shape
    assert bool(((out.double() - ref).abs() <= bound).all())


def test_moe_layer_row_without_local_experts_is_zero():
    c = MoECase(T=8, H=64, E=8, k=1, inner=64, first=7, local=1)
    out = ops.moe_layer(*c.args())
    chosen = torch.softmax(c.x.float() @ c.router.float().t(), -1).argmax(-1)
    assert bool((out[chosen != 7] == 0).all())


def test_refusals():
    x = torch.zeros(2, 10)
    tok = torch.zeros(2, dtype=torch.int64)
    for bad in (lambda: ops.token_logprobs(x, tok, top=33), lambda: ops.token_logprobs(x, tok, top=-1),
                lambda: ops.token_logprobs(x, tok[:1]), lambda: ops.token_logprobs(x, tok.float()),
                lambda: ops.token_logprobs(x, tok[None])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        ops.token_logprobs(x.half(), tok)
    h, w = torch.zeros(2, 16).bfloat16(), torch.zeros(10, 16).bfloat16()
    with pytest.raises(ValueError):
        ops.linear_logprobs(h, w[:, :8], tok)
    for cap in (-1.0, INF, NAN):
        with pytest.raises(ValueError):
            ops.linear_logprobs(h, w, tok, softcap=cap)
    with pytest.raises(TypeError):
        ops.linear_logprobs(h, [w], tok)
    c = MoECase(T=2, H=64, E=4, k=2, inner=64)
    a = list(c.args())

    def but(**kw):
        b = dict(enumerate(a))
        b.update({int(i[1:]): v for i, v in kw.items()})
        return [b[i] for i in range(len(a))]

    for bad in (but(_0=torch.zeros(17, 64).bfloat16()), but(_3=100), but(_5=63), but(_6=0), but(_6=5),
                but(_4=a[4][:-1]), but(_8=1), but(_8=-1)):
        with pytest.raises(ValueError):
            ops.moe_layer(*bad)


def test_softcap_whose_reciprocal_fp32_cannot_hold():
    h, w, tok = torch.zeros(2, 16).bfloat16(), torch.zeros(10, 16).bfloat16(), torch.zeros(2, dtype=torch.int64)
    for cap in (1e-300, 1e-45, 1e-39, 1e39, 1e300):
        with pytest.raises(ValueError, match="softcap"):
            ops.linear_logprobs(h, w, tok, softcap=cap)
    for cap in (0, 2.0 ** -100, 2.0 ** 100):
        assert all(bool(t.isfinite().all()) for t in ops.linear_logprobs(h, w, tok, softcap=cap))

"""LM-head scoring at the sizes and with the options that users run: the error that its split sums are for, tiles of
two CTAs with capped logits, hidden sizes that leave a part and a block unfilled, a whole vocabulary."""

import math

import pytest
import torch

from b200serve import ops
from logprob_cases import INF, check_linear_logprobs

pytestmark = pytest.mark.gpu
dev = "cuda"


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)
    ops.ext()


def _stats64(x, w, tokens):
    """In 64 bits, on the GPU: log probability, entropy, the logits' root mean square and largest spread in a row."""
    logits = torch.cat([x.double() @ p.double().t() for p in w.split(16384)], 1)
    logp = torch.log_softmax(logits, -1)
    return (logp.gather(1, tokens[:, None])[:, 0], -(logp.exp() * logp).sum(-1), logits.pow(2).mean().sqrt().item(),
            logits.std(-1).max().item())


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("T", [100, 300])
def test_error_of_the_split_sums(packed, T):
    """Root-mean-square error of the log probabilities at H = 4096 beside that of the logits.

    The tensor cores cut each addition of 16 products, by half a last place of the running sum on average and always
    towards zero: after n of them a sum of size r is off by about n 2^-24 (2/3) r. In parts of 512 elements
    n = 32 and r = sqrt(512 / 4096) of the logit; eight parts of either sign make 32 * 2^-24 * 2/3 * 0.354 * sqrt(8) =
    1.3e-6 of the logit (less for shorter parts). A log probability takes two such logits, the token's and, where one dominates, the
    largest: sqrt 2 of it, 1.8e-6. One sum over H would have n = 256: 1.0e-5 for a logit, 1.4e-5."""
    H, V = 4096, 320
    x = torch.randn(T, H, device=dev).bfloat16()
    w = (torch.randn(V, H, device=dev) * 8.0 / math.sqrt(H)).bfloat16()       # logits of root mean square 8
    tokens = torch.randint(0, V, (T,), device=dev)
    want, _, rms, _ = _stats64(x, w, tokens)
    lp, _ = ops.linear_logprobs(x, ops.PackedWeight(w) if packed else w, tokens)
    err = (lp.double() - want).pow(2).mean().sqrt().item()
    assert 6 < rms < 10 and err < 2e-6 * rms, (err / rms)


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("T", [5, 129, 200, 300])
def test_softcap_and_unfilled_parts(packed, T):
    """H = 1608 is 26 blocks of 64, the last one of 8: parts of 4 or 8 blocks with a remainder of 2. T > 128 takes two
    CTAs per tile."""
    V, H = 3001, 1608
    w = (torch.randn(V, H, device=dev) * 20.0 / math.sqrt(H)).bfloat16()
    x = torch.randn(T, H, device=dev).bfloat16()
    tokens = torch.randint(0, V, (T,), device=dev)
    head = ops.PackedWeight(w) if packed else w
    for cap in (0.0, 15.0):
        check_linear_logprobs(ops.linear_logprobs(x, head, tokens, softcap=cap), x, w, tokens, cap)
    assert ops.linear_logprobs_error() == 0


@pytest.mark.parametrize("T", [1, 23, 700])
def test_a_whole_vocabulary(T):
    """151936 tokens of 4096 elements. Per logit the parts above leave 1.3e-6 of its size, so 5 times that for the
    largest of T * V (their errors are sums of many terms); the entropy's derivative is bounded by 2 ln V, and the sums
    over V add the bounds of the shared statistics."""
    from logprob_cases import entropy_bound, logprob_bound
    V, H = 151936, 4096
    w = (torch.randn(V, H, device=dev) * 1.3 / math.sqrt(H)).bfloat16()
    tokens = torch.randint(0, V, (T,), device=dev)
    x = (torch.randn(T, H, device=dev) + torch.rand(T, 1, device=dev) * 8 * w[tokens].float()).bfloat16()
    want, ent, _, spread = _stats64(x, w, tokens)
    logit_err = 5 * 1.3e-6 * max(spread, 16.0)               # the token's own logit reaches 8 * 1.3^2 + 3
    lp, en = ops.linear_logprobs(x, ops.PackedWeight(w), tokens)
    assert float((lp.double() - want).abs().max()) < logprob_bound(V, float(want.abs().max()), logit_err)
    assert float((en.double() - ent).abs().max()) < entropy_bound(V, logit_err)
    two = ops.token_logprobs(ops.linear(x, ops.PackedWeight(w), epilogue=ops.EPI_F32), tokens)
    # linear() keeps one sum over H: 1.0e-5 of a logit on average
    assert float((lp - two.logprob).abs().max()) < 5 * 2 * 1.0e-5 * 16.0


def test_few_rows_are_as_exact_as_a_rounded_product():
    """Up to 128 rows take parts of 128 elements. As above, 8 cuts leave 8 * 2^-24 * 2/3 * sqrt(128 / 4096) = 5.6e-8 of the
    logit, sqrt(32) times that over 32 parts of either sign: 3.2e-7; the 32 rounded additions of a growing sum leave
    2^-24 / sqrt 3 * sqrt(32 / 3) = 1.1e-7. Together 3.4e-7, sqrt 2 of it for the two logits that count: 4.8e-7 (with a
    last place of 2^-23 throughout, its upper end). Parts of 256 elements measure 5.4e-7, of 128 3.6e-7."""
    H, V, T = 4096, 64, 128
    w = (torch.randn(V, H, device=dev) * 8.0 / math.sqrt(H)).bfloat16()
    x = torch.randn(T, H, device=dev).bfloat16()
    tokens = torch.randint(0, V, (T,), device=dev)
    want, _, rms, _ = _stats64(x, w, tokens)
    err = torch.cat([ops.linear_logprobs(x[i:i + 1], w, tokens[i:i + 1])[0] for i in range(T)]).double() - want
    assert err.pow(2).mean().sqrt().item() < 4.8e-7 * rms
    lp, _ = ops.linear_logprobs(x, w, tokens)
    assert (lp.double() - want).pow(2).mean().sqrt().item() < 4.8e-7 * rms


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("T", [1, 40, 200, 1000])
def test_likely_tokens(packed, T):
    """Rows that lean towards their token: the products of its logit (4 to 16) are mostly positive, so that cuts would all
    go one way. log p = -log1p(r), r = sum e^(x_j - x_token) over thousands of small terms whose own errors cancel; what
    moves all of them is the token's logit: half a last place of it (below 16) 4.8e-7, its sum of 8-element chains and a
    tree a third of that (1.6e-7, independent), and ex2's bias, at most 2^-22 = 2.4e-7: 7.5e-7 of log p. Left out:
    rows with another leader (log p is a difference of logits then, with that one's error) and logits from 16 on."""
    V, H = 6000, 4096
    w = (torch.randn(V, H, device=dev) * 1.3 / math.sqrt(H)).bfloat16()
    tokens = torch.randint(0, V, (T,), device=dev)
    lift = torch.linspace(11.5, 15, T, device=dev)[:, None] / 1.69
    x = (torch.randn(T, H, device=dev) * 0.5 + lift * w[tokens].float()).bfloat16()
    z = x.double() @ w.double().t()
    top = z.gather(1, tokens[:, None])[:, 0]
    d = (z - top[:, None]).scatter_(1, tokens[:, None], -INF)
    rest = d.exp().sum(-1)
    lead = (d.amax(-1) < 0) & (top < 16)
    want, ent = -torch.log1p(rest), torch.log1p(rest) - (d.exp() * d.clamp_min(-1e30)).sum(-1) / (1 + rest)
    lp, en = ops.linear_logprobs(x, ops.PackedWeight(w) if packed else w, tokens)
    rel = ((lp.double() - want) / want)[lead]
    assert float(lead.float().mean()) > 0.9
    assert rel.pow(2).mean().sqrt().item() < 7.5e-7
    # the entropy's terms carry d e^d: twice as much
    assert (((en.double() - ent) / ent)[lead]).pow(2).mean().sqrt().item() < 1.5e-6

"""Log-probability kernels at the edges of their inputs' range, against 64-bit references."""

import math

import pytest
import torch

from b200serve import ops
from logprob_cases import check_token_logprobs, entropy_bound, log_s_bound

pytestmark = pytest.mark.gpu
dev = "cuda"


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)
    ops.ext()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_whole_slices_at_the_lowest_value(dtype):
    """Rows masked with the type's lowest value instead of -inf, whole slices of 8192 logits among them."""
    V, low = 30001, torch.finfo(dtype).min
    x = torch.randn(5, V, device=dev)
    x[0, 8192:] = low
    x[1, 100:29000] = low
    x[2, :29000] = low
    x[3] = low                                           # all of it: a uniform distribution
    x[4, 9000:] = low
    x[4, 3] = 3e38                                       # differences past the largest float
    x = x.to(dtype)
    tokens = torch.tensor([5, 29500, 7, 12000, 3], device=dev)
    check_token_logprobs(ops.token_logprobs(x, tokens, top=20), x, tokens, 20)


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("T", [2, 200])
def test_logits_far_below_zero(packed, T):
    """Every logit of a row below -1e30: what pads a tile past the vocabulary must not count. 300 and 40 tokens
    leave the last tile part empty; the 2^100s are exact, and differ by 0 or by 2^100."""
    for V in (300, 40):
        x = torch.zeros(T, 64, device=dev, dtype=torch.bfloat16)
        w = torch.zeros(V, 64, device=dev, dtype=torch.bfloat16)
        x[:, 0], w[:, 0] = 1, -(2.0 ** 101)
        tokens = torch.full((T,), 7, device=dev)
        head = ops.PackedWeight(w) if packed else w
        lp, ent = ops.linear_logprobs(x, head, tokens)
        want = math.log(V)                               # uniform
        assert float((lp + want).abs().max()) < log_s_bound(V) + want * 2.0 ** -22
        assert float((ent - want).abs().max()) < entropy_bound(V)
        w[9, 0] = -(2.0 ** 100)                          # one token takes everything
        head = ops.PackedWeight(w) if packed else w
        lp, ent = ops.linear_logprobs(x, head, tokens)
        assert bool((lp == -(2.0 ** 100)).all() and (ent == 0).all())
        tokens[:] = 9
        assert bool((ops.linear_logprobs(x, head, tokens)[0] == 0).all())


def test_results_are_void_until_the_error_word_is_read():
    """After a bounded wait has run out (here: its code is put into the error word) no plausible numbers come back."""
    x, w = torch.randn(5, 64, device=dev).bfloat16(), torch.randn(500, 64, device=dev).bfloat16()
    tokens = torch.arange(5, device=dev)
    good = ops.linear_logprobs(x, w, tokens)
    assert ops.ext().linear_logprobs_error(13) == 0
    void = ops.linear_logprobs(x, w, tokens)
    assert all(bool(t.isnan().all()) for t in void)
    assert ops.linear_logprobs_error(reset=False) == 13 and ops.linear_logprobs_error() == 13
    assert ops.linear_logprobs_error() == 0
    assert all(torch.equal(a, b) for a, b in zip(good, ops.linear_logprobs(x, w, tokens)))


def test_softcap_at_the_ends_of_its_range():
    x, w = torch.randn(9, 64, device=dev).bfloat16(), torch.randn(500, 64, device=dev).bfloat16()
    tokens = torch.arange(9, device=dev)
    got, plain = ops.linear_logprobs(x, w, tokens, softcap=2.0 ** 100), ops.linear_logprobs(x, w, tokens)
    assert all(torch.equal(a, b) for a, b in zip(got, plain))            # powers of two: the same bits
    lp, ent = ops.linear_logprobs(x, w, tokens, softcap=2.0 ** -100)     # every logit next to 0: uniform
    want = math.log(500)
    assert float((lp + want).abs().max()) < log_s_bound(500) + want * 2.0 ** -22
    assert float((ent - want).abs().max()) < entropy_bound(500)


def test_rows_that_overlap_in_memory():
    """x.expand() and windows of one buffer: legal strides, and every row is what indexing says."""
    w = torch.randn(700, 128, device=dev).bfloat16()
    buf = torch.randn(4096, device=dev).bfloat16()
    for T in (5, 150):
        tokens = torch.randint(0, 700, (T,), device=dev)
        for x in (buf[:128].expand(T, -1), buf.as_strided((T, 128), (8, 1)), buf.as_strided((T, 128), (4, 1))):
            got, want = ops.linear_logprobs(x, w, tokens), ops.linear_logprobs(x.clone().contiguous(), w, tokens)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


# Log probabilities of almost certain tokens: -log1p(r), r = sum of the others' e^d. A term is off by ex2's (or, joining
# slices, __expf's) 2^-21 and the rounding of d and d log2(e), 2^-23 |d| with |d| <= 40 here; the sums add 80 * 2^-24, log1p 2^-23:
# 2^-21 + 40 * 2^-23 + 80 * 2^-24 + 2^-23 < 1.1e-5 of the value. Beside the 1 of a whole sum only 2^-24 = 6e-8 absolute is left.
_CERTAIN = 1.1e-5


def _certain_rows(V, n):
    g = torch.Generator(device=dev).manual_seed(7)
    x = torch.randn(n, V, device=dev, generator=g)
    peak = torch.randint(0, V, (n,), device=dev, generator=g)
    x[torch.arange(n, device=dev), peak] = torch.linspace(12, 38, n, device=dev)
    return x, peak


def _check_certain(lp, ent, logits, tokens):
    d = logits.double() - logits.double().amax(-1, keepdim=True)
    own = torch.zeros_like(d, dtype=torch.bool).scatter_(1, tokens[:, None], True)
    e = d.exp().masked_fill(own, 0.0)
    rest = e.sum(-1)
    want = -torch.log1p(rest)
    entropy = torch.log1p(rest) - (e * d).sum(-1) / (1 + rest)
    assert float(want.abs().min()) < 1e-9 and float(want.abs().max()) > 0.02
    assert float(((lp.double() - want) / want).abs().max()) < _CERTAIN
    assert float(((ent.double() - entropy) / entropy).abs().max()) < 2 * _CERTAIN      # t carries the error of d as well


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [3000, 50001])
def test_almost_certain_tokens(dtype, V):
    x, peak = _certain_rows(V, 60)
    x = x.to(dtype)
    got = ops.token_logprobs(x, peak, top=2)
    _check_certain(got.logprob, got.entropy, x, peak)
    assert torch.equal(got.top_logprobs[:, 0], got.logprob) and torch.equal(got.top_ids[:, 0], peak.int())


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("T", [1, 60, 200])
def test_almost_certain_tokens_of_the_head(packed, T):
    """One-hot rows, so that the logits are the head's own bf16 numbers."""
    V, H = 5000, 256
    x, peak = _certain_rows(V, H)
    w = x.t().contiguous().bfloat16()                                    # column h: the logits of the one-hot row h
    rows = torch.linspace(0, H - 1, T, device=dev).long() if T > 1 else torch.tensor([H - 1], device=dev)
    hot = torch.eye(H, device=dev).bfloat16()[rows]
    lp, ent = ops.linear_logprobs(hot, ops.PackedWeight(w) if packed else w, peak[rows])
    if T == 1:
        assert -1e-9 < lp.item() < 0 and 0 < ent.item() < 1e-7
    else:
        _check_certain(lp, ent, w.float().t()[rows], peak[rows])

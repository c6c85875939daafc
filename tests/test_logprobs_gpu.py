"""Log-probability kernels against 64-bit references: sizes from one entry up, strided and misaligned rows, ties,
masks, rows without a distribution, streams and graphs."""

import pytest
import torch

from b200serve import ops
from logprob_cases import INF, NAN, check_linear_logprobs, check_token_logprobs

pytestmark = pytest.mark.gpu
dev = "cuda"


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)
    ops.ext()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,V,top", [(1, 1, 1), (1, 3, 5), (2, 17, 17), (3, 4096, 20), (5, 4097, 32), (4, 8193, 1),
                                     (2, 32003, 20), (1, 151936, 20), (20, 32000, 5), (300, 1000, 3), (2, 50257, 0)])
def test_token_logprobs(dtype, B, V, top):
    x = (torch.randn(B, V, device=dev) * 3).to(dtype)
    tokens = torch.randint(0, V, (B,), device=dev)
    check_token_logprobs(ops.token_logprobs(x, tokens, top=top), x, tokens, top)
    tokens[:] = x.float().argmax(-1)
    got = ops.token_logprobs(x, tokens.int(), top=top)
    check_token_logprobs(got, x, tokens, top)
    if top:
        assert torch.equal(got.top_logprobs[:, 0], got.logprob)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("skip", [0, 1, 3])
def test_token_logprobs_strided_and_misaligned(dtype, skip):
    buf = (torch.randn(6, 9003, device=dev) * 3).to(dtype)
    x = buf[:, skip:skip + 8999]
    tokens = torch.tensor([0, 8998, 1, 4095, 4096, 77], device=dev)
    check_token_logprobs(ops.token_logprobs(x, tokens, top=20), x, tokens, 20)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_logprobs_ties(dtype):
    V = 20011
    x = torch.zeros(6, V, device=dev)                                   # all equal: the lowest ids
    x[1] = torch.arange(V, device=dev).float()                          # ascending (many ties in bf16)
    x[2] = -torch.arange(V, device=dev).float()
    x[3] = torch.randint(0, 4, (V,), device=dev).float()                # a few values
    x[4, ::2] = -0.0                                                    # signed zeros are equal
    x[5] = -INF
    x[5, 19990:] = torch.finfo(dtype).min                               # the type's lowest value is a logit
    x = x.to(dtype)
    tokens = torch.tensor([10000, 3, V - 1, 5, 1, 20000], device=dev)
    for top in (1, 20, 32):
        check_token_logprobs(ops.token_logprobs(x, tokens, top=top), x, tokens, top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_logprobs_masks_and_rows_without_a_distribution(dtype):
    V = 30001
    x = torch.randn(9, V, device=dev)
    x[0, torch.rand(V, device=dev) < 0.999] = -INF
    x[1] = -INF                                                         # nothing left
    x[2] = -INF
    x[2, 29000] = 1.5                                                   # one entry left: log probability 0
    x[3, 12345] = NAN
    x[4, 0] = INF
    x[5] = NAN
    x[6, :8192] = -INF                                                  # a whole slice masked
    x[7] *= 1e4                                                         # one token takes everything
    x = x.to(dtype)
    tokens = torch.tensor([5, 0, 29000, 1, 0, 2, 100, int(x[7].float().argmax()), V], device=dev)
    check_token_logprobs(ops.token_logprobs(x, tokens, top=20), x, tokens, 20)
    tokens[:] = -1
    check_token_logprobs(ops.token_logprobs(x, tokens, top=2), x, tokens, 2)


def test_token_logprobs_empty_batch_and_wide_vocabulary():
    got = ops.token_logprobs(torch.empty(0, 50, device=dev), torch.empty(0, dtype=torch.int64, device=dev), top=3)
    assert got.logprob.shape == (0,) and got.top_ids.shape == (0, 3)
    x = torch.randn(2, 1 << 20, device=dev)
    tokens = torch.tensor([(1 << 20) - 1, 0], device=dev)
    check_token_logprobs(ops.token_logprobs(x, tokens, top=32), x, tokens, 32)


def test_token_logprobs_rows_past_32_bits():
    V, rows = 1 << 20, 2 * 2049
    buf = torch.zeros(rows, V, dtype=torch.bfloat16, device=dev)         # 4.3 G elements
    x = buf[::2048]                                                     # rows 2^31 elements apart
    x.copy_(torch.randn(x.shape[0], V, device=dev))
    tokens = torch.full((x.shape[0],), V - 7, device=dev)
    check_token_logprobs(ops.token_logprobs(x, tokens, top=8), x, tokens, 8)


def _linear_case(T, V, H, scale=1.3):
    w = (torch.randn(V, H, device=dev) * scale / H ** 0.5).bfloat16()
    tokens = torch.randint(0, V, (T,), device=dev)
    x = (torch.randn(T, H, device=dev) + torch.rand(T, 1, device=dev) * 6 * w[tokens].float()).bfloat16()
    return x, w, tokens


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("T,V,H", [(1, 1, 8), (1, 1000, 64), (3, 127, 72), (1, 32000, 256), (127, 129, 200), (128, 4096, 64),
                                   (129, 5003, 136), (300, 32000, 256), (1, 40001, 1024), (513, 1000, 4096)])
def test_linear_logprobs(packed, T, V, H):
    x, w, tokens = _linear_case(T, V, H)
    got = ops.linear_logprobs(x, ops.PackedWeight(w) if packed else w, tokens)
    check_linear_logprobs(got, x, w, tokens, 0.0)
    assert ops.linear_logprobs_error() == 0


@pytest.mark.parametrize("T", [2, 70])
def test_linear_logprobs_softcap_and_unknown_tokens(T):
    x, w, tokens = _linear_case(T, 3001, 264, scale=20.0)               # logits far past the cap
    tokens[0], tokens[1] = -1, 3001
    check_linear_logprobs(ops.linear_logprobs(x, w, tokens, softcap=15.0), x, w, tokens, 15.0)
    check_linear_logprobs(ops.linear_logprobs(x, ops.PackedWeight(w), tokens.int()), x, w, tokens, 0.0)


def test_linear_logprobs_bad_rows_stay_alone():
    x, w, tokens = _linear_case(130, 2000, 128)
    good = ops.linear_logprobs(x, w, tokens)
    x[5, 3], x[64, 0], x[129, 127] = NAN, INF, -INF
    got = ops.linear_logprobs(x, w, tokens)
    keep = torch.ones(130, dtype=torch.bool, device=dev)
    keep[[5, 64, 129]] = False
    for a, b in zip(got, good):
        assert torch.equal(a[keep], b[keep]) and bool(a[~keep].isnan().all())


def test_linear_logprobs_strided_rows_and_more_than_one_pass():
    x, w, tokens = _linear_case(9000, 300, 64)                          # 8192 rows a pass
    wide = torch.zeros(9000, 96, device=dev, dtype=torch.bfloat16)
    wide[:, 16:80] = x
    got = ops.linear_logprobs(wide[:, 16:80], w, tokens)
    check_linear_logprobs([t[8100:8300] for t in got], x[8100:8300], w, tokens[8100:8300], 0.0)
    again = ops.linear_logprobs(x, w, tokens)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_linear_logprobs_agrees_with_the_logits_path():
    """The same rows through linear() + token_logprobs, as a prompt's alternatives are computed."""
    x, w, tokens = _linear_case(40, 32000, 256)
    pw = ops.PackedWeight(w)
    lp, ent = ops.linear_logprobs(x, pw, tokens)
    two = ops.token_logprobs(ops.linear(x, pw, epilogue=ops.EPI_F32), tokens, top=5)
    assert float((lp - two.logprob).abs().max()) < 1e-4 and float((ent - two.entropy).abs().max()) < 1e-3


def test_streams_graphs_and_repeats():
    x, w, tokens = _linear_case(50, 5000, 192)
    logits = x.float() @ w.float().t()
    want = ops.token_logprobs(logits, tokens, top=7), ops.linear_logprobs(x, w, tokens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.token_logprobs(logits, tokens, top=7), ops.linear_logprobs(x, w, tokens)
    here = ops.token_logprobs(logits, tokens, top=7), ops.linear_logprobs(x, w, tokens)   # both streams at once
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        in1 = ops.token_logprobs(logits, tokens, top=7), ops.linear_logprobs(x, w, tokens)
    with torch.cuda.graph(g2):
        in2 = ops.token_logprobs(logits, tokens, top=7), ops.linear_logprobs(x, w, tokens)
    for _ in range(3):
        g1.replay()
        g2.replay()
    torch.cuda.synchronize()
    for got in (other, here, in1, in2):
        for a, b in zip(got, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_refusals_on_the_gpu():
    x = torch.zeros(2, 64, device=dev)
    tok = torch.zeros(2, dtype=torch.int64, device=dev)
    h, w = x.bfloat16(), torch.zeros(10, 64, device=dev).bfloat16()
    for bad in (lambda: ops.token_logprobs(x, tok.cpu()), lambda: ops.token_logprobs(x.t()[:2], tok),
                lambda: ops.token_logprobs(torch.zeros(2, (1 << 20) + 1, device=dev), tok),
                lambda: ops.linear_logprobs(x, w, tok), lambda: ops.linear_logprobs(h, w.float(), tok),
                lambda: ops.linear_logprobs(h, w.cpu(), tok), lambda: ops.linear_logprobs(h[:, 1:33], w[:, :32], tok),
                lambda: ops.linear_logprobs(h[:, :60], w[:, :60].contiguous(), tok),
                lambda: ops.linear_logprobs(h.t()[:2, :2], w[:, :2].contiguous(), tok)):
        with pytest.raises((RuntimeError, ValueError)):
            bad()

"""Log-probability kernels at the edges of their inputs' range, against 64-bit references."""

import pytest
import torch

from b200serve import ops
from logprob_cases import check_token_logprobs

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

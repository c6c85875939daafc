"""The small-batch MoE layer where something is wrong: a wait that runs out, weights and activations out of range."""

import pytest
import torch

from b200serve import ops
from logprob_cases import INF, NAN, MoECase

pytestmark = pytest.mark.gpu
dev = "cuda"


@pytest.fixture(autouse=True)
def _ext():
    ops.ext()


def test_a_wait_that_runs_out_is_reported_and_its_outputs_are_void():
    """A gate/up unit reads 16 rows of 262144 elements (8 MB), far longer than 64 looks at the counter take, so with a
    limit of a microsecond the other CTAs give up; all of it ends by itself."""
    c = MoECase(T=1, H=262144, E=1, k=1, inner=64)
    a = c.args(dev)
    want = ops.moe_layer(*a)
    assert ops.moe_layer_error() == 0 and not bool(want.isnan().any())
    old = ops.ext().get_flag_wait_ms()
    try:
        ops.ext().set_flag_wait_ms(0.001)
        out = ops.moe_layer(*a)
    finally:
        ops.ext().set_flag_wait_ms(old)
    assert ops.moe_layer_error(reset=False) == 24 and ops.moe_layer_error(wait=False) == 24
    assert bool(out.isnan().any())
    assert bool((out.isnan() | (out == want)).all())         # void or right, nothing in between
    assert ops.moe_layer_error() == 0
    assert torch.equal(ops.moe_layer(*a), want) and ops.moe_layer_error() == 0

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


@pytest.mark.parametrize("T", [3, 8, 16])
@pytest.mark.parametrize("value", [INF, NAN])
def test_an_experts_bad_weight_reaches_only_its_own_tokens(T, value):
    c = MoECase(T=T, H=128, E=16, k=2, inner=96)
    a = list(c.args(dev))
    good = ops.moe_layer(*a)
    z = c.router.double() @ c.x.double().t()
    chosen = z.topk(c.k, dim=0).indices                      # [k, T]
    tiles = a[4].shape[0] // c.E
    for e in sorted(set(chosen.flatten().tolist()))[:4]:
        bad = list(a)
        bad[4] = a[4].clone()
        bad[4][e * tiles + 3, 5] = value                     # down row 3, inner column 5
        got = ops.moe_layer(*bad)
        own = (chosen == e).any(0).to(dev)
        keep = torch.ones(T, c.H, dtype=torch.bool, device=dev)
        keep[own, 3] = False
        assert torch.equal(got[keep], good[keep]) and not bool(got[own, 3].isfinite().any())
        bad[4] = a[4]
        bad[2] = a[2].clone()
        bad[2][e * (a[2].shape[0] // c.E) + 3, 5] = value    # gate row 3 of the expert
        got = ops.moe_layer(*bad)
        assert torch.equal(got[~own], good[~own]) and not bool(got[own].isfinite().all(-1).any())

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


@pytest.mark.parametrize("T", [1, 6, 16])
@pytest.mark.parametrize("up", [1.4140625 * 2.0 ** 64, -1.4140625 * 2.0 ** 64, 2.0 ** 90, -2.0 ** 90])
def test_activations_at_the_end_of_the_range(T, up):
    """silu(1.4140625 * 2^63) * up: +-1.99957 * 2^127 lies between bf16's largest value and fp32's (the output is
    exact to bf16's rounding), with 2^90 it is +-infinity (the output has the down weight's sign)."""
    c = MoECase(T=T, H=64, E=1, k=1, inner=1)
    g = torch.Generator().manual_seed(1)
    c.x.zero_()
    c.x[:, 0] = 1.0
    size = torch.randint(64, 128, (c.H,), generator=g) * 2.0 ** -17          # 8-bit factors of 2^-11 to 2^-10
    down = (size * torch.where(torch.rand(c.H, generator=g) < 0.5, -1.0, 1.0)).bfloat16()
    a = list(c.args(dev))
    tiles_gu, tiles_dn = torch.zeros_like(a[2]), torch.zeros_like(a[4])
    tiles_gu[0, 0], tiles_gu[64, 0] = 1.4140625 * 2.0 ** 63, up              # gate row 0, up row 0
    tiles_dn[:c.H, 0] = down.to(dev)
    a[2], a[4] = tiles_gu, tiles_dn
    act = torch.tensor(1.4140625 * 2.0 ** 63, dtype=torch.float64) * up
    if abs(up) == 2.0 ** 90:
        act = act.sign() * INF
    want = (act * down.double()).bfloat16().expand(T, -1)
    assert torch.equal(ops.moe_layer(*a).cpu(), want)


@pytest.mark.parametrize("T", [1, 16])
def test_a_router_written_by_the_kernel_before(T):
    """The router is an operand like the rows: a kernel right before the call, which lets the next one start early,
    may write it."""
    c = MoECase(T=T, H=2048, E=32, k=4, inner=64)
    a = list(c.args(dev))
    g = torch.Generator(device=dev).manual_seed(3)
    sources = [torch.randn(32, 2048, device=dev, generator=g).bfloat16() for _ in range(6)]
    scale = torch.full((2048,), 0.03, device=dev, dtype=torch.bfloat16)
    want = []
    for s in sources:
        a[1] = ops.rmsnorm(s, scale, 1e-6).clone()
        torch.cuda.synchronize()
        want.append(ops.moe_layer(*a))
    a[1] = torch.zeros(32, 2048, device=dev, dtype=torch.bfloat16)

    def passes():
        out = []
        for s in sources:
            ops.rmsnorm(s, scale, 1e-6, out=a[1])
            out.append(ops.moe_layer(*a))
        return out

    eager = passes()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = passes()
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    for outs in (eager, captured):
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_out_may_be_x_and_its_rows_may_not_overlap():
    c = MoECase(T=9, H=256, E=12, k=3, inner=96)
    a = list(c.args(dev))
    want = ops.moe_layer(*a)
    for bad in (torch.empty(1, 256, device=dev).bfloat16().expand(9, -1),
                torch.empty(4096, device=dev).bfloat16().as_strided((9, 256), (128, 1))):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.moe_layer(*a, out=bad)
    same = a[0] = a[0].clone()
    assert ops.moe_layer(*a, out=same) is same and torch.equal(same, want)


_FIRST_CALL = """
import sys
sys.path[:0] = ["tests", "."]
import torch
from b200serve import ops
from logprob_cases import MoECase
c = MoECase(T=5, H=256, E=8, k=2, inner=64)
a = c.args("cuda")
x, w, t = torch.randn(5, 64, device="cuda").bfloat16(), torch.randn(300, 64, device="cuda").bfloat16(), \\
    torch.arange(5, device="cuda")
ops.ext()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out, (lp, ent) = ops.moe_layer(*a), ops.linear_logprobs(x, w, t)
    tok = ops.token_logprobs(x.float(), t, top=3)
g.replay()
torch.cuda.synchronize()
ref, bound = c.reference()
assert bool(((out.double().cpu() - ref).abs() <= bound).all()) and ops.moe_layer_error() == 0
assert all(torch.equal(p, q) for p, q in zip((lp, ent), ops.linear_logprobs(x, w, t)))
assert all(torch.equal(p, q) for p, q in zip(tok, ops.token_logprobs(x.float(), t, top=3)))
print("captured")
"""


def test_the_first_call_of_a_process_may_be_captured():
    """What a process sets up once (the error words, the kernels' attributes) is allowed inside a capture."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _FIRST_CALL], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]

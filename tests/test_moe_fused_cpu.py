"""When EngineConfig.moe_fused takes effect (MoEBlock.use_fused), on the CPU."""

import logging
from types import SimpleNamespace

import pytest
import torch

from b200serve import ops
from b200serve.models.config import BUILTIN
from b200serve.models.moe import MoEBlock


def _block(comm=None, **cfg):
    mc = BUILTIN["tiny-qwen3-moe"]
    for k, v in cfg.items():
        mc = type(mc)(**{**vars(mc), k: v})
    router = ops.PackedWeight(torch.randn(mc.num_experts, mc.hidden_size).bfloat16())
    weights = SimpleNamespace(layers=[SimpleNamespace(router=router) for _ in range(2)], ep_size=1, ep_rank=0)
    return MoEBlock(mc, weights, comm=comm, device="cpu")


class _Fused:                                        # the fused communicator's face to the block
    max_tokens = 64

    def moe_combine_reduce(self, y, wts, pos, k, T):
        raise AssertionError("not called")


def test_use_fused_copies_the_routers():
    for comm in (None, SimpleNamespace(world=2)):
        b = _block(comm)
        assert b.use_fused() is True and b.fused_rows == ops.MOE_LAYER_MAX_ROWS
        assert all(torch.equal(b.routers[i], lw.router.unpacked()) for i, lw in enumerate(b.w.layers))


def test_fused_communicator_keeps_its_own_combine(caplog):
    b = _block(_Fused())
    with caplog.at_level(logging.WARNING):
        assert b.use_fused() is False
    assert "moe_fused is off" in caplog.text and b.routers == {} and b.fused_rows == 0


@pytest.mark.parametrize("cfg,on", [(dict(num_experts=512), False), (dict(num_experts=256), True),
                                    (dict(num_experts=32, experts_per_tok=17), False)])
def test_models_past_the_layers_limits_keep_the_grouped_path(cfg, on, caplog):
    b = _block(**cfg)
    with caplog.at_level(logging.WARNING):
        assert b.use_fused() is on
    assert ("moe_fused is off" in caplog.text) != on and bool(b.routers) == on and bool(b.fused_rows) == on

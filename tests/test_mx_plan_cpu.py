"""Plans rewritten for microscaled weights."""
import pytest

from tinyinfer_b200.config.registry import architecture_of
from tinyinfer_b200.parts.microscaled import MxAttention, MxPreNormBlock, MxRMSNorm, MxSwiGLU, microscaled_plan
from tinyinfer_b200.parts.model import CausalLM

import kagorax_util
from util import TINY


def plan_of(cfg):
    arch = architecture_of(cfg)
    return arch.build_plan(arch.from_dict(cfg))


@pytest.mark.parametrize("name", sorted(TINY))
def test_layers_get_microscaled_parts_and_the_same_tensors(name):
    plan = plan_of(TINY[name])
    model, plain = CausalLM(microscaled_plan(plan, "mxfp4")), CausalLM(plan)
    for block in model.blocks:
        assert type(block) is MxPreNormBlock and type(block.mixer) is MxAttention and type(block.ffn) is MxSwiGLU
        assert type(block.mixer_norm) is type(block.ffn_norm) is MxRMSNorm
    assert model.expected_tensors() == plain.expected_tensors() and model.cache_specs() == plain.cache_specs()


def test_other_layers_and_formats_are_refused():
    with pytest.raises(ValueError, match="no such form"):
        microscaled_plan(plan_of(kagorax_util.SMALL["C"][0]), "mxfp4")
    with pytest.raises(ValueError, match="must be one of"):
        microscaled_plan(plan_of(TINY["A"]), "int4")


def test_float32_engines_refuse_the_format():
    from tinyinfer_b200 import Engine
    with pytest.raises(ValueError, match="bfloat16"):
        Engine(config=TINY["A"], seed=1, dtype="float32", weights="mxfp4", ops=object())

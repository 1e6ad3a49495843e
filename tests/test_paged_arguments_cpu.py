"""Arguments of the attention programs that have to be refused, and what a refusal leaves behind."""
import math

import pytest

import intent_b200 as ib


@pytest.mark.parametrize("program", ["paged_attention", "paged_decode_attention"])
@pytest.mark.parametrize("scale", [1e-46, 1e-300, 1e39, 0, -0.0, -1e-3, math.inf, math.nan, "a"])
def test_scales_that_are_no_positive_f32(program, scale):
    """One that is zero as f32 is not the default of 1 / sqrt(D)."""
    with pytest.raises(ib.CompilationStageError):
        ib.compile(getattr(ib.programs, program), constexprs={"SCALE": scale}, resolve_target=False)


@pytest.mark.parametrize("scale", [None, 1e-45, 0.125, 1, 3e38])
def test_scales_that_are_one(scale):
    artifact = ib.compile(ib.programs.paged_attention, constexprs={"SCALE": scale}, resolve_target=False)
    assert (artifact.runtime.constants[0] == 0) == (scale is None)

"""The example of the 8-bit cache's operators: rounds of prefill, verification, commit, decode.

P is rounded to bf16 (2^-8), exp2 is within 2^-12, the output is rounded to bf16 (2^-8 of
|out| <= sum w |v|): below 2^-6 of sum w |v| with room for the queries' and fp32 sums' terms.
"""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sizes", [dict(), dict(requests=7, kv_heads=2, groups=7, dim=64, block=16,
                                                longest=300, nodes=16, seed=3)])
def test_rounds_agree_with_fp32_attention(sizes):
    path = Path(__file__).resolve().parents[1] / "examples" / "fp8_verify_rounds.py"
    spec = importlib.util.spec_from_file_location("fp8_verify_rounds", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    worst, state = module.main(**sizes)
    assert worst < 2.0 ** -6
    assert (state.cached > 0).all()

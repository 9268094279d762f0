"""How near the half-width outputs of the delta rule come to the exact ones.

The error of a result rounded from x + d is that of the rounding, uniform in its step and independent of d, and d: their squares add.  |d| is
1e-5 |x| for sums in fp32 (test_delta_rule.py); under bfloat16 the operands of o have 16 bits, each of the three that meet (S or P, U
and the product's dropped terms) 2^-17 off at most: 2.3e-5 more."""
import numpy as np
import pytest
import torch

from test_delta_rule import SUM, TYPES, args, inputs, oracle, rel


@pytest.mark.gpu
@pytest.mark.parametrize("kind,extra", [("f16", 0.0), ("bf16", 3 * 2.0 ** -17)])
@pytest.mark.parametrize("B,T,Hk,Hv,dk,dv", [(1, 300, 2, 2, 64, 32), (2, 500, 1, 2, 128, 128), (1, 1000, 1, 1, 100, 40)])
def test_outputs_are_as_near_as_rounding_allows(B, T, Hk, Hv, dk, dv, kind, extra):
    from gaussian_process_amd import gated_delta_rule
    x = inputs(B, T, Hk, Hv, dk, dv, kind, seed=1, slow=True)
    want = oracle(*args(x), x["state"])[0]
    rounding = rel(torch.tensor(want).to(TYPES[kind]), want)
    o = gated_delta_rule(*args(x), initial_state=x["state"])[0]
    assert rel(o, want) <= np.hypot(rounding, SUM + extra)

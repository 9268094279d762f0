"""The gradient of the log decay, head by head: heads that forget quickly have small ones, which one norm over all heads hides.

Every term of d_g at a token carries the token's own exp(g), so that the relative error does not depend on g.  Terms are products of
four sums in fp32 over at most 128 + 64 terms (1e-5, as in test_delta_rule.py); they have random signs and add up to about the root of the
sum of their squares, ten times less at worst here: 1e-4 of the norm over a head's tokens."""
import numpy as np
import pytest
import torch

from test_delta_rule import TYPES, args, cu, inputs, oracle

TOL = 1e-4
RATES = (-0.01, -1.0, -4.0, -8.0, -12.0, -16.0)


def fast_heads(x):
    rates = torch.tensor(RATES, device="cuda")
    x["g"].copy_(rates * (0.8 + 0.4 * torch.rand(x["g"].shape, generator=torch.Generator().manual_seed(1)).cuda()))
    return x


def gradients(x, kind, offsets=None):
    from gaussian_process_amd import gated_delta_rule, gated_delta_rule_backward
    rng = np.random.default_rng(2)
    d_o = torch.tensor(rng.standard_normal(x["v"].shape)).to(TYPES[kind]).cuda()
    d_f = torch.tensor(rng.standard_normal(x["state"].shape)).float().cuda()
    c = None if offsets is None else cu(offsets)
    saved = gated_delta_rule(*args(x), initial_state=x["state"], cu_seqlens=c, save_for_backward=True)[2]
    got = gated_delta_rule_backward(saved, d_o, d_f)[3]
    return got.double().cpu().numpy(), oracle(*args(x), x["state"], offsets, None, d_o, d_f)[5]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("B,T,Hk,dk,dv", [(1, 200, 6, 64, 32), (2, 130, 2, 128, 40), (13, 200, 3, 100, 16), (44, 17, 2, 48, 16), (1, 3, 6, 16, 8)])
def test_every_head(B, T, Hk, dk, dv, kind):
    """Key heads alone, value heads on workgroups of their own, and (more than 256 chunks) one after the other."""
    got, want = gradients(fast_heads(inputs(B, T, Hk, 6, dk, dv, kind, seed=T)), kind)
    for h, rate in enumerate(RATES):
        err = np.linalg.norm(got[..., h] - want[..., h]) / np.linalg.norm(want[..., h])
        assert err < TOL, (rate, err)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_packed(kind):
    off = [0, 0, 1, 64, 66, 200, 331]
    got, want = gradients(fast_heads(inputs(1, 331, 3, 6, 64, 32, kind, seqs=6, seed=4)), kind, off)
    for h, rate in enumerate(RATES):
        err = np.linalg.norm(got[..., h] - want[..., h]) / np.linalg.norm(want[..., h])
        assert err < TOL, (rate, err)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_nothing_behind_a_reset(kind):
    """exp(-infinity) = 0: what a reset token forgets has no gradient, and its own g none at all."""
    x = inputs(1, 150, 1, 6, 64, 32, kind)
    at = (0, 1, 15, 16, 40, 63, 64, 100, 149)
    x["g"][:, at] = -float("inf")
    got, want = gradients(x, kind)
    assert (got[:, at] == 0).all() and (want[:, at] == 0).all() and np.isfinite(got).all()
    assert np.linalg.norm(got - want) < TOL * np.linalg.norm(want)

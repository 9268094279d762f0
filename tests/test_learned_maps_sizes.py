"""Sizes at the ends of what the learned maps take: beyond 32 bits refused (and not cut off), the largest stack computed."""
import pytest
import torch


def big(*shape, dtype=torch.float32):
    return torch.zeros(1, dtype=dtype).expand(shape)   # no memory


@pytest.mark.parametrize("what", ["tokens", "batch", "heads"])
@pytest.mark.parametrize("n", [(1 << 32) + 64, (1 << 31) + 1, (1 << 30) + 1])
def test_delta_sizes_beyond_32_bits(what, n):
    from gaussian_process_amd import gated_delta_rule, gated_delta_rule_step
    B, T, H = (n if what == w else 1 for w in ("batch", "tokens", "heads"))
    with pytest.raises(ValueError, match="2\\^30"):
        gated_delta_rule(big(B, T, H, 4), big(B, T, H, 4), big(B, T, H, 4), big(B, T, H), big(B, T, H))
    if what != "tokens":
        with pytest.raises(ValueError, match="2\\^30"):
            gated_delta_rule_step(big(B, H, 4), big(B, H, 4), big(B, H, 4), big(B, H), big(B, H), big(B, H, 4, 4))


def test_sequences_and_states_beyond_32_bits():
    from gaussian_process_amd import gated_delta_rule, gated_delta_rule_step
    row = [torch.zeros(1, 1, 1, 4)] * 3 + [torch.zeros(1, 1, 1)] * 2
    with pytest.raises(ValueError, match="too many"):
        gated_delta_rule(*row, cu_seqlens=big((1 << 32) + 3, dtype=torch.int32))
    with pytest.raises(ValueError, match="too many"):
        gated_delta_rule_step(*(t[:, 0] for t in row), big((1 << 32) + 1, 1, 4, 4), slots=torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("shape", [((1 << 32) + 2, 4, 4), (1 << 17, 1 << 15, 4, 4), ((1 << 32) + 2, 4), (4, (1 << 32) + 2), (65537, 4)])
def test_orthogonalize_sizes_beyond(shape):
    from gaussian_process_amd import orthogonalize
    with pytest.raises(ValueError, match="more than"):
        orthogonalize(big(*shape))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["float64", "float32", "bfloat16"])
def test_the_largest_stack(kind):
    from gaussian_process_amd import _lib, orthogonalize
    from test_orthogonalize import TOL, plain
    G = torch.randn(65535, 3, 2, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(getattr(torch, kind))
    # one step: 40 u hold where no direction is far below the others, which small matrices do not keep to
    O = orthogonalize(G, steps=1).double().cpu()
    want = torch.tensor(plain(G, steps=1))
    err = ((O - want).square().sum((1, 2)) / want.square().sum((1, 2))).sqrt()
    assert err.max().item() < TOL[{"float64": "f64", "float32": "f32", "bfloat16": "bf16"}[kind]]
    with pytest.raises(_lib.GpxError):
        orthogonalize(torch.zeros(65536, 1, 1, device="cuda"))

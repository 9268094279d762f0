"""Single tokens on states at any address: part of a pool whose states are of odd sizes, or of a larger buffer."""
import pytest
import torch


def row(B, Hk, Hv, dk, dv, device="cpu"):
    g = torch.Generator().manual_seed(dk)
    x = [torch.randn(B, Hk, dk, generator=g), torch.randn(B, Hk, dk, generator=g) * dk ** -0.5, torch.randn(B, Hv, dv, generator=g),
         -torch.rand(B, Hv, generator=g), torch.rand(B, Hv, generator=g)]
    return [t.to(device) for t in x]


def shifted(t, n):
    """t's values n elements behind a 16-byte boundary."""
    buf = torch.zeros(t.numel() + 4 + n, dtype=t.dtype, device=t.device)
    assert buf.data_ptr() % 16 == 0
    out = buf[n:n + t.numel()].view(t.shape)
    return out.copy_(t), buf


def test_not_refused_for_its_address():
    from gaussian_process_amd import _lib, gated_delta_rule_step
    pool = torch.zeros(4, 1, 5, 5)
    assert pool[1:].data_ptr() % 16 != 0
    with pytest.raises(_lib.GpxError, match="MI355X"):   # as far as a call gets without a GPU
        gated_delta_rule_step(*row(3, 1, 1, 5, 5), pool[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("dk,dv", [(5, 5), (64, 64), (100, 12), (128, 130)])
@pytest.mark.parametrize("n,m", [(1, 0), (0, 1), (2, 3), (3, 3)])
def test_same_as_aligned(dk, dv, n, m):
    from gaussian_process_amd import gated_delta_rule_step
    x = row(3, 1, 2, dk, dv, "cuda")
    state = torch.randn(3, 2, dk, dv, device="cuda")
    want_o, want = gated_delta_rule_step(*x, state, state_out=torch.empty_like(state))
    a, buf_a = shifted(state, n)
    b, buf_b = shifted(torch.zeros_like(state), m)
    o, _ = gated_delta_rule_step(*x, a, state_out=b)
    assert torch.equal(o, want_o) and torch.equal(b, want) and torch.equal(a, state)
    assert (buf_b[:m] == 0).all() and (buf_b[m + b.numel():] == 0).all()   # nothing beside it
    slots = torch.tensor([2, -1, 0], dtype=torch.int32, device="cuda")
    c = state.clone()
    o1, _ = gated_delta_rule_step(*x, c, slots=slots)
    o2, _ = gated_delta_rule_step(*x, a, slots=slots)
    assert torch.equal(o1, o2) and torch.equal(a, c) and (buf_a[:n] == 0).all() and (buf_a[n + a.numel():] == 0).all()

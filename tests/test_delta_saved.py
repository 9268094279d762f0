"""What a saving forward call of the delta rule keeps: the memory of its inputs, whatever the caller does with the tensors."""
import ctypes as C
import gc

import pytest
import torch


def host_saved():
    from gaussian_process_amd import _lib, delta
    x = [torch.randn(1, 70, 1, 8), torch.randn(1, 70, 1, 8), torch.randn(1, 70, 2, 8), torch.randn(1, 70, 2), torch.randn(1, 70, 2)]
    d = _lib.Delta(1, 1, 70, 0, 1, 2, 8, 8, 1.0, None, *(t.data_ptr() for t in x))
    return x, d, delta.Saved(d, x, None, torch.empty(256, dtype=torch.uint8), None)


def test_memory_is_kept_when_a_tensor_is_given_another():
    x, d, saved = host_saved()
    want = [t.clone() for t in x]
    names = ("q", "k", "v", "g", "beta")
    for t in x:
        t.data = torch.full_like(t, 7.0)
    del x, t
    gc.collect()
    again = [torch.full((1 << 12,), 9.0) for _ in range(64)]   # noqa: F841  (what freed memory would be given to)
    for name, kept, value in zip(names, saved.inputs, want):
        assert kept.data_ptr() == getattr(d, name)
        held = torch.frombuffer((C.c_float * value.numel()).from_address(getattr(d, name)), dtype=torch.float32)
        assert torch.equal(held.view(value.shape), value)
    saved.check()


@pytest.mark.parametrize("i", range(5))
def test_resized_storage_is_refused(i):
    from gaussian_process_amd import gated_delta_rule_backward
    x, d, saved = host_saved()
    saved.check()
    x[i].untyped_storage().resize_(0)
    with pytest.raises(RuntimeError, match="resized"):
        gated_delta_rule_backward(saved, torch.zeros(1, 70, 2, 8))


@pytest.mark.parametrize("i", range(5))
def test_writes_are_refused(i):
    from gaussian_process_amd import gated_delta_rule_backward
    x, d, saved = host_saved()
    x[i][:, :1].add_(1.0)
    with pytest.raises(RuntimeError, match="modified"):
        gated_delta_rule_backward(saved, torch.zeros(1, 70, 2, 8))


@pytest.mark.gpu
def test_gradients_after_a_tensor_is_given_another():
    from gaussian_process_amd import gated_delta_rule, gated_delta_rule_backward
    torch.manual_seed(0)
    x = [torch.randn(2, 200, 2, 64, device="cuda").bfloat16() * 0.1 for _ in range(2)]
    x += [torch.randn(2, 200, 2, 32, device="cuda").bfloat16(), -torch.rand(2, 200, 2, device="cuda"), torch.rand(2, 200, 2, device="cuda")]
    d_o = torch.randn_like(x[2])
    saved = gated_delta_rule(*x, save_for_backward=True)[2]
    want = gated_delta_rule_backward(saved, d_o)[:5]
    for t in x:
        t.data = torch.zeros_like(t)
    nan = [torch.full_like(t, float("nan")) for t in x for _ in range(4)]   # noqa: F841  (into the memory, were it free)
    assert all(torch.equal(a, b) for a, b in zip(want, gated_delta_rule_backward(saved, d_o)))
    with pytest.raises(RuntimeError):
        saved.inputs[1].untyped_storage().resize_(0)
        gated_delta_rule_backward(saved, d_o)

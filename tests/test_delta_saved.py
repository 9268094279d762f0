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


def _ranges(tensors):
    return [(t.data_ptr(), t.data_ptr() + t.untyped_storage().nbytes()) for t in tensors]


@pytest.mark.gpu
def test_memory_is_kept_for_another_stream():
    """The saved values are dropped while a backward call on another stream has yet to read them: their memory is not handed out before
    that stream is done.  The control shows that the allocator does hand it out where nothing waits."""
    from gaussian_process_amd import gated_delta_rule, gated_delta_rule_backward
    torch.manual_seed(1)
    B, T, H, d = 1, 4096, 8, 64
    x = [0.1 * torch.randn(B, T, d, H, device="cuda").transpose(2, 3) for _ in range(2)]   # not dense: saved holds copies
    x += [torch.randn(B, T, H, d, device="cuda"), -torch.rand(B, T, H, device="cuda"), torch.rand(B, T, H, device="cuda")]
    d_o = torch.randn(B, T, H, d, device="cuda")
    big = torch.randn(8192, 8192, device="cuda")
    product = torch.empty_like(big)

    def forward():
        saved = gated_delta_rule(*x, save_for_backward=True)[2]
        own = [saved.work, *saved.inputs[:2]]
        assert saved.inputs[0].data_ptr() != x[0].data_ptr()
        return saved, _ranges(own), [t.untyped_storage().nbytes() for t in own]

    def handed_out(old, sizes):
        new = _ranges([torch.empty(n, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(3)])
        return any(a < d and c < b for a, b in old for c, d in new)

    want = gated_delta_rule_backward(forward()[0], d_o)
    _, old, sizes = forward()
    torch.cuda.synchronize()
    del _
    assert handed_out(old, sizes)
    saved, old, sizes = forward()
    side, done = torch.cuda.Stream(), torch.cuda.Event()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(8):
            torch.mm(big, big, out=product)   # some 10 ms each
        got = gated_delta_rule_backward(saved, d_o)
        done.record()
    del saved
    early = handed_out(old, sizes)
    assert not done.query(), "the other stream was done before the test looked"
    assert not early
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got) if a is not None)

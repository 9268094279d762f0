"""The learned maps record no gradient: a call that would lose one is refused before it does anything."""
import pytest
import torch
from torch.autograd import forward_ad


def calls():
    """Each entry point with its tensors by name."""
    from gaussian_process_amd import _lib, gated_delta_rule, gated_delta_rule_backward, gated_delta_rule_step, orthogonalize
    from gaussian_process_amd.delta import Saved
    x = dict(q=torch.zeros(1, 5, 1, 4), k=torch.zeros(1, 5, 1, 4), v=torch.zeros(1, 5, 2, 3), g=torch.zeros(1, 5, 2), beta=torch.zeros(1, 5, 2))
    row = {n: t[:, 0].clone() for n, t in x.items()}
    state = torch.zeros(1, 2, 4, 3)
    d = _lib.Delta(1, 1, 5, 0, 1, 2, 4, 3)
    saved = Saved(d, list(x.values()), None, torch.empty(256, dtype=torch.uint8), None)
    yield gated_delta_rule, dict(x, initial_state=state)
    yield lambda **kw: gated_delta_rule_backward(saved, **kw), dict(d_o=x["v"], d_final_state=state)
    yield gated_delta_rule_step, dict(row, state=state)
    yield gated_delta_rule_step, dict(row, state=state, state_out=state.clone())
    W = torch.zeros(4, 6)
    yield lambda **kw: orthogonalize(beta=0.5, **kw), dict(G=W, base=W.clone(), out=W.clone())


CASES = [(i, name) for i, (_, kw) in enumerate(calls()) for name in kw]


@pytest.mark.parametrize("i,name", CASES)
def test_refused_where_torch_records(i, name):
    from gaussian_process_amd import _lib
    call, kw = list(calls())[i]
    kw[name] = kw[name].detach().requires_grad_()
    with pytest.raises(RuntimeError, match="gradient"):
        call(**kw)
    with torch.no_grad(), pytest.raises(_lib.GpxError, match="MI355X"):   # as far as a call gets without a GPU
        call(**kw)
    kw[name] = kw[name] * 1   # not a leaf
    with pytest.raises(RuntimeError, match="gradient"):
        call(**kw)
    kw[name] = kw[name].detach()
    with pytest.raises(_lib.GpxError, match="MI355X"):
        call(**kw)


@pytest.mark.parametrize("i,name", CASES)
def test_tangents_are_refused(i, name):
    from gaussian_process_amd import _lib
    call, kw = list(calls())[i]
    with forward_ad.dual_level():
        with pytest.raises(_lib.GpxError, match="MI355X"):
            call(**kw)
        kw[name] = forward_ad.make_dual(kw[name], torch.ones_like(kw[name]))
        with pytest.raises(RuntimeError, match="tangent"):
            call(**kw)


@pytest.mark.gpu
def test_parameters_under_no_grad():
    """An optimiser's update and a decoder's step write what requires a gradient where torch would too."""
    from gaussian_process_amd import gated_delta_rule_step, orthogonalize
    W = torch.nn.Parameter(torch.randn(40, 60, device="cuda"))
    G, before = torch.randn_like(W), W.detach().clone()
    with pytest.raises(RuntimeError, match="gradient"):
        orthogonalize(G, alpha=-0.1, beta=0.9, base=W, out=W)
    assert torch.equal(W.detach(), before)
    with torch.no_grad():
        orthogonalize(G, alpha=-0.1, beta=0.9, base=W, out=W)
    assert torch.equal(W.detach(), orthogonalize(G, alpha=-0.1, beta=0.9, base=before))
    row = [torch.randn(2, h, 8, device="cuda") for h in (1, 1, 2)] + [-torch.rand(2, 2, device="cuda"), torch.rand(2, 2, device="cuda")]
    state = torch.zeros(2, 2, 8, 8, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="gradient"):
        gated_delta_rule_step(*row, state)
    assert (state == 0).all()
    with torch.inference_mode():
        gated_delta_rule_step(*row, state)
    assert (state != 0).any()

"""How near bfloat16 results of orthogonalize come: by default as near as rounding allows, with reduced=True in 11 bits.

A result round(x + d) with |d| <= D, x the exact one, is within |round(x) - x| + 2 |d| of x, element by element, so that its error in
the 2-norm is that of rounding the exact result plus 2 D.  D = 40 * 2^-22 |x| as for float32 (test_orthogonalize.py).  reduced: D = 40 * 2^-12 |x|,
the tolerance of one fp16 value per intermediate."""
import ctypes as C

import numpy as np
import pytest
import torch

from test_orthogonalize import make, plain, rel

SHAPES = [(1, 1), (16, 40), (130, 260), (300, 100), (512, 512), (3, 200, 520), (700, 1300), (64, 4000)]


def rounding(x):
    return rel(torch.tensor(x).bfloat16(), x)


def test_refused_for_other_types():
    from gaussian_process_amd import orthogonalize
    for t in (torch.float16, torch.float32, torch.float64):
        with pytest.raises(ValueError, match="reduced"):
            orthogonalize(torch.zeros(4, 6, dtype=t), reduced=True)


def test_work_bytes_of_two_planes():
    from gaussian_process_amd import _lib
    w = _lib.load().gpx_orthogonalize_work_bytes
    for sizes in ((1, 65, 130), (3, 700, 300), (1, 256, 4096)):
        assert w(3 | _lib.GPX_TWO_PLANES, *sizes) == w(2, *sizes) > w(3, *sizes)
    for other in (0, 1, 2, 4):
        assert w(other | _lib.GPX_TWO_PLANES, 1, 65, 130) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_default_is_as_near_as_rounding_allows(shape):
    from gaussian_process_amd import orthogonalize
    G = make(shape, "bf16", seed=3)
    want = plain(G)
    assert rel(orthogonalize(G), want) <= rounding(want) + 2 * 40 * 2.0 ** -22
    W = make(shape, "bf16", seed=4, scale=0.3)
    want = 0.9 * W.double().cpu().numpy() - 0.1 * want
    assert rel(orthogonalize(G, alpha=-0.1, beta=0.9, base=W), want) <= rounding(want) + 2 * 40 * 2.0 ** -22


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_reduced(shape):
    from gaussian_process_amd import orthogonalize
    G = make(shape, "bf16", seed=3)
    want = plain(G)
    O = orthogonalize(G, reduced=True)
    assert rel(O, want) <= rounding(want) + 2 * 40 * 2.0 ** -12
    assert torch.equal(O, orthogonalize(G, reduced=True))
    W = make(shape, "bf16", seed=4, scale=0.3)
    V = W.clone()
    orthogonalize(G, alpha=-0.1, beta=0.9, base=V, out=V, reduced=True)
    want = 0.9 * W.double().cpu().numpy() - 0.1 * want
    assert rel(V, want) <= rounding(want) + 2 * 40 * 2.0 ** -12


@pytest.mark.gpu
def test_reduced_stacks_views_zeros_and_not_finite():
    from gaussian_process_amd import orthogonalize
    big = make((2, 90, 140), "bf16", seed=4)
    for G in (big[0].mT, big[:, 3:80, 5:110], big[:, ::2, ::3], big.permute(2, 0, 1), big.mT[:, 1:, 1:]):
        want = plain(G)
        assert rel(orthogonalize(G, reduced=True), want) <= rounding(want) + 2 * 40 * 2.0 ** -12
    G = make((3, 70, 90), "bf16")
    want = plain(G[:1])
    G[1] = 0
    G[2, 5, 6] = float("nan")
    O = orthogonalize(G, reduced=True)
    assert rel(O[:1], want) <= rounding(want) + 2 * 40 * 2.0 ** -12 and (O[1] == 0).all() and O[2].isnan().all()


@pytest.mark.gpu
def test_library_refuses_the_flag_for_other_types():
    from gaussian_process_amd import _lib
    from gaussian_process_amd.device import runtime
    rt = runtime()
    buf = torch.zeros(1 << 16, device="cuda")
    st, coef = _lib.Strided(0, 8, 1), (C.c_double * 3)(3.4445, -4.7750, 2.0315)
    for other in (0, 1, 2, 4):
        with rt.current_stream():
            rc = rt.lib.gpx_orthogonalize(rt.h, other | _lib.GPX_TWO_PLANES, 1, 8, 8, buf.data_ptr(), C.byref(st), 5, coef, 1e-7, 1.0, 0.0, None, None,
                                          buf.data_ptr(), C.byref(st), buf.data_ptr(), buf.numel() * 4)
        assert rc == -1
    assert (buf == 0).all() and np.isfinite(buf.cpu().numpy()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16", "f64"])
@pytest.mark.parametrize("coef,steps", [((0.5, 0.0, 0.0), 13), ((0.25, -0.1, 0.02), 8), ((0.1, 0.3, 0.0), 5)])
def test_coefficients_that_shrink(kind, coef, steps):
    """The spectrum's bound falls by the polynomial's factor at every step, and the intermediates' scale goes with it: the tolerance of
    test_orthogonalize.py.  Results down to 1e-4 are normal numbers of every type once alpha has brought them back."""
    from gaussian_process_amd import orthogonalize
    from test_orthogonalize import TOL
    G = make((72, 200), kind, seed=steps)
    want = plain(G, steps, coef) / coef[0] ** steps
    got = orthogonalize(G, steps=steps, coefficients=coef, alpha=coef[0] ** -steps)
    assert rel(got, want) < TOL[kind], rel(got, want)
    if kind == "f32":   # far down; alpha is not needed there
        want = plain(G, 4 * steps, coef)
        assert rel(orthogonalize(G, steps=4 * steps, coefficients=coef), want) < TOL[kind]

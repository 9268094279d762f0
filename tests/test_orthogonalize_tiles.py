"""orthogonalize on every tile that its products are formed in, half (X X^T, A A) and whole (B X), with sides that end inside a tile; against
the definition in 64 bits, with the tolerances of test_orthogonalize.py."""
import pytest
import torch

from test_orthogonalize import COEF, TOL, TYPES

SHAPES = [(40, 190, 288), (64, 280, 287), (40, 616, 280), (16, 550, 1210), (40, 640, 647), (8, 1300, 777), (1, 4060, 4067)]
KINDS = ["f32", "f16", "bf16", "reduced"]


def tiles(kind, shape):
    from gaussian_process_amd import _lib
    dtype = {"f32": 1, "f16": 2, "bf16": 3 | _lib.GPX_TWO_PLANES, "reduced": 3}[kind]
    return [_lib.load().gpx_orthogonalize_tile(dtype, *shape, product) for product in range(3)]


@pytest.mark.parametrize("kind", KINDS)
def test_every_tile_is_reached(kind):
    """So that a rule that chooses otherwise takes nothing out of the test below: half products in tiles of 128, 192 and 256, whole ones too,
    each with a padded side (a multiple of 64) that is none of the tile's."""
    reached = set()
    for shape in SHAPES:
        n, m = ((x + 63) // 64 * 64 for x in sorted(shape[1:]))
        for product, tile in enumerate(tiles(kind, shape)):
            if n % tile or (product == 2 and m % tile):
                reached.add((product == 2, tile))
    assert reached == {(whole, tile) for whole in (False, True) for tile in (128, 192, 256)}
    assert tiles(kind, (1, 100, 200)) == [64, 64, 64]   # the sizes of test_orthogonalize.py


def test_tile_of_refused_calls():
    from gaussian_process_amd import _lib
    f = _lib.load().gpx_orthogonalize_tile
    assert f(0, 1, 100, 100, 0) == f(1, 0, 100, 100, 0) == f(1, 1, 0, 100, 0) == f(1, 1, 100, 100, 3) == f(9, 1, 100, 100, 0) == 0


def plain(G):
    X = G.double()
    flip = X.shape[-2] > X.shape[-1]
    X = X.mT.contiguous() if flip else X
    X = X / (X.square().sum((-2, -1), keepdim=True).sqrt() + 1e-7)
    for _ in range(5):
        A = X @ X.mT.contiguous()
        X = COEF[0] * X + (COEF[1] * A + COEF[2] * (A @ A)) @ X
    return X.mT if flip else X


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_the_definition(shape, kind):
    from gaussian_process_amd import orthogonalize
    reduced = kind == "reduced"
    t = TYPES["bf16" if reduced else kind]
    g = torch.Generator(device="cuda").manual_seed(shape[1])
    G = (1e-3 * torch.randn(shape, generator=g, device="cuda")).to(t)
    W = torch.randn(shape, generator=g, device="cuda").to(t)
    want = plain(G)
    O = orthogonalize(G, reduced=reduced)
    per = lambda x: x.square().sum((-2, -1)).sqrt()   # noqa: E731
    tol = TOL["bf16" if reduced else kind]
    assert (per(O.double() - want) / per(want)).max().item() < tol
    into = torch.zeros(shape[0], shape[2], shape[1], dtype=t, device="cuda").mT   # written along columns
    orthogonalize(G, alpha=-0.5, beta=0.75, base=W, out=into, reduced=reduced)
    want = 0.75 * W.double() - 0.5 * want
    assert (per(into.double() - want) / per(want)).max().item() < tol

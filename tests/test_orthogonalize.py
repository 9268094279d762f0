"""gaussian_process_amd.orthogonalize against its definition in 64 bits.

Tolerances, relative in the 2-norm.  u is half a step of what an intermediate is held in (fp64 2^-53, pairs of fp16
2^-22, one fp16 2^-11); every step rounds X, A and B once and multiplies three times, and an error in the direction of a
singular value s/40 of the largest counts 40 times more there, hence 40 u; the result's own rounding (2^-8 bf16, 2^-11
fp16, 2^-24 fp32) comes on top.  The random matrices here have few directions below 1/40 of the largest."""
import numpy as np
import pytest
import torch

COEF = (3.4445, -4.7750, 2.0315)
TYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TOL = {"f64": 40 * 2.0 ** -53 * 8, "f32": 40 * 2.0 ** -22 + 2.0 ** -24, "f16": 40 * 2.0 ** -22 + 2.0 ** -11,
       "bf16": 40 * 2.0 ** -12 + 2.0 ** -8}


def plain(G, steps=5, coef=COEF, eps=1e-7):
    X = np.asarray(G.double().cpu())
    flip = X.shape[-2] > X.shape[-1]
    X = np.swapaxes(X, -1, -2) if flip else X
    X = X / (np.sqrt((X * X).sum((-2, -1), keepdims=True)) + eps)
    for _ in range(steps):
        A = X @ np.swapaxes(X, -1, -2)
        X = coef[0] * X + (coef[1] * A + coef[2] * A @ A) @ X
    return np.swapaxes(X, -1, -2) if flip else X


def rel(a, b):
    a = a.double().cpu().numpy()
    return np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-300)


# ---- refusals (no GPU) --------------------------------------------------------------------------------------------
def test_refusals():
    from gaussian_process_amd import _lib, orthogonalize
    G = torch.zeros(4, 6)
    with pytest.raises(_lib.GpxError):
        orthogonalize(G)
    with pytest.raises(TypeError):
        orthogonalize(np.zeros((4, 6)))
    with pytest.raises(TypeError):
        orthogonalize(G.int())
    with pytest.raises(ValueError):
        orthogonalize(G[0])
    with pytest.raises(ValueError):
        orthogonalize(G, beta=0.5)
    with pytest.raises(ValueError):
        orthogonalize(G, beta=0.5, base=torch.zeros(6, 4))
    with pytest.raises(ValueError):
        orthogonalize(G, out=torch.zeros(4, 6, dtype=torch.float64))
    with pytest.raises(ValueError):
        orthogonalize(G, coefficients=(1.0, 2.0))
    with pytest.raises(ValueError):
        orthogonalize(G, out=torch.zeros(1, 6).expand(4, 6))


def test_work_bytes():
    from gaussian_process_amd import _lib
    lib = _lib.load()
    for dtype, planes in ((1, 2), (2, 2), (3, 1)):
        assert lib.gpx_orthogonalize_work_bytes(dtype, 3, 65, 130) == 3 * (8192 + 2 * ((4 + 2 * planes) * 128 * 192 + 2 * planes * 128 * 128))
        assert lib.gpx_orthogonalize_work_bytes(dtype, 1, 130, 65) == lib.gpx_orthogonalize_work_bytes(dtype, 1, 65, 130)
    assert lib.gpx_orthogonalize_work_bytes(0, 1, 5, 40) == 8192 + 8 * (2 * 32 * 64 + 2 * 5 * 32)
    assert lib.gpx_orthogonalize_work_bytes(9, 1, 5, 40) == 0
    assert lib.gpx_orthogonalize_work_bytes(1, 1, 0, 40) == 0
    # a long K split over workgroups: room for the parts' sums
    whole = 8192 + 2 * (8 * 256 * 4096 + 4 * 256 * 256)
    assert (lib.gpx_orthogonalize_work_bytes(1, 1, 256, 4096) - whole) % (256 * 256 * 4) == 0
    assert lib.gpx_orthogonalize_work_bytes(1, 1, 256, 4096) > whole
    # 64-bit sizes
    assert lib.gpx_orthogonalize_work_bytes(1, 1, 65536, 65536) == 8192 + 2 * 12 * 65536 ** 2


# ---- GPU ----------------------------------------------------------------------------------------------------------
def make(shape, kind, seed=0, scale=1e-3):
    rng = np.random.default_rng(seed)
    return torch.tensor(scale * rng.standard_normal(shape)).to(TYPES[kind]).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (9, 1), (16, 40), (64, 128), (63, 65), (200, 130), (128, 512), (257, 390),
                                   (3, 40, 100), (2, 2, 70, 33)])
def test_matches_the_definition(shape, kind):
    from gaussian_process_amd import orthogonalize
    G = make(shape, kind, seed=len(shape) + shape[-1])
    O = orthogonalize(G)
    assert O.shape == G.shape and O.dtype == G.dtype
    ref = plain(G)
    assert rel(O, ref) < TOL[kind], rel(O, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", [(100, 3000), (2, 260, 4100), (2600, 640), (3, 64, 8000), (333, 1001), (3, 200, 520), (700, 300)])
def test_long_rows(shape, kind):
    """Few tiles of a long K, which fp64 and two planes split over workgroups."""
    from gaussian_process_amd import orthogonalize
    G = make(shape, kind, seed=shape[-1])
    O = orthogonalize(G)
    assert rel(O, plain(G)) < TOL[kind]
    assert torch.equal(O, orthogonalize(G))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_singular_values(kind):
    from gaussian_process_amd import orthogonalize
    s = np.linalg.svd(orthogonalize(make((150, 600), kind)).double().cpu().numpy(), compute_uv=False)
    assert 0.6 < s.min() and s.max() < 1.25


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("steps,coef", [(1, COEF), (2, COEF), (12, (1.5, -0.5, 0.0)), (3, (2.0, -1.5, 0.5))])
def test_steps_and_coefficients(steps, coef, kind):
    from gaussian_process_amd import orthogonalize
    G = make((72, 200), kind, seed=steps)
    ref = plain(G, steps, coef)
    assert rel(orthogonalize(G, steps=steps, coefficients=coef), ref) < TOL[kind]


@pytest.mark.gpu
def test_eps_shrinks_a_small_matrix():
    from gaussian_process_amd import orthogonalize
    G = make((20, 30), "f32", scale=1e-9)
    ref = plain(G, steps=2)
    assert rel(orthogonalize(G, steps=2), ref) < TOL["f32"]
    # squares of these underflow in 32 bits
    G = make((20, 30), "f32", scale=1e-30)
    assert rel(orthogonalize(G, eps=0.0), plain(G, eps=0.0)) < TOL["f32"]
    G = make((20, 30), "f32", scale=1e30)
    assert rel(orthogonalize(G), plain(G)) < TOL["f32"]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_zeros_and_not_finite(kind):
    from gaussian_process_amd import orthogonalize
    G = make((3, 70, 90), kind)
    ref = plain(G)
    G[1] = 0
    G[2, 5, 6] = float("nan")
    O = orthogonalize(G)
    assert rel(O[0], ref[0]) < TOL[kind]       # a stack's matrices do not touch each other
    assert (O[1] == 0).all()
    assert O[2].isnan().all()
    G[2, 5, 6] = float("inf")
    assert orthogonalize(G)[2].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_views_and_strides(kind):
    from gaussian_process_amd import orthogonalize
    big = make((2, 90, 140), kind, seed=4)
    for G in (big[0].mT, big[:, 3:80, 5:110], big[:, ::2, ::3], big.permute(2, 0, 1), big[0, :1].expand(40, 140),
              big.mT[:, 1:, 1:]):
        assert rel(orthogonalize(G), plain(G)) < TOL[kind]
        into = torch.full_like(big.new_empty(*G.shape[:-2], 2 * G.shape[-1], G.shape[-2] + 3), 7.0)
        out = into.mT[..., 3:, ::2] if G.dim() == 2 or G.shape[0] == 2 else torch.empty_like(G)
        before = into.clone()
        O = orthogonalize(G, out=out)
        assert O is out and rel(out, plain(G)) < TOL[kind]
        if out.untyped_storage().data_ptr() == into.untyped_storage().data_ptr():
            assert (into[..., 1::2, :] == before[..., 1::2, :]).all() and (into[..., :3] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", [(65, 130), (130, 65), (2, 30, 30)])
def test_update_in_place(shape, kind):
    from gaussian_process_amd import orthogonalize
    G, W = make(shape, kind, 1), make(shape, kind, 2, scale=0.3)
    want = 0.9 * W.double().cpu().numpy() - 0.1 * plain(G)
    there = orthogonalize(G, alpha=-0.1, beta=0.9, base=W)
    assert rel(there, want) < TOL[kind]
    V = W.clone()
    assert orthogonalize(G, alpha=-0.1, beta=0.9, base=V, out=V) is V
    assert torch.equal(V, there)
    # out over G
    H = G.clone()
    orthogonalize(H, alpha=-0.1, beta=0.9, base=W, out=H)
    assert torch.equal(H, there)
    # base is another view of out's memory
    if shape[-1] == shape[-2]:
        V = W.clone()
        orthogonalize(G, alpha=-0.1, beta=0.9, base=V.mT, out=V)
        assert rel(V, 0.9 * W.mT.double().cpu().numpy() - 0.1 * plain(G)) < TOL[kind]
    # beta = 0 does not read base
    assert torch.equal(orthogonalize(G, base=torch.full_like(G, float("nan"))), orthogonalize(G))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_out_over_a_shifted_stack(kind):
    """out one matrix behind G in the same memory, and G's matrices in the opposite order."""
    from gaussian_process_amd import orthogonalize
    buf = make((4, 20, 33), kind, seed=8)
    want = orthogonalize(buf[:3].clone())
    assert torch.equal(orthogonalize(buf[:3], out=buf[1:]), want) and torch.equal(buf[1:], want)
    G = make((33, 33), kind, seed=9)
    want = orthogonalize(G.clone().mT)
    assert torch.equal(orthogonalize(G.mT, out=G), want)


@pytest.mark.gpu
def test_empty():
    from gaussian_process_amd import orthogonalize
    for shape in ((0, 5), (5, 0), (0, 4, 4)):
        assert orthogonalize(torch.zeros(shape, device="cuda")).shape == shape


@pytest.mark.gpu
def test_refused_by_the_library():
    from gaussian_process_amd import _lib, orthogonalize
    G = make((8, 8), "f32")
    for bad in (dict(steps=0), dict(steps=65), dict(coefficients=(10.0, 10.0, 10.0)), dict(coefficients=(float("nan"), 0, 0)),
                dict(eps=-1.0), dict(eps=float("nan")), dict(alpha=float("inf"))):
        with pytest.raises(_lib.GpxError):
            orthogonalize(G, **bad)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_streams_and_graphs(kind):
    """Two calls at once on two streams; two captured graphs with their own workspaces, replayed in turn with eager
    work between; nothing depends on what ran before."""
    from gaussian_process_amd import orthogonalize
    Gs = [make((130, 260), kind, seed) for seed in (1, 2)]
    want = [orthogonalize(G) for G in Gs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in Gs]
    got = []
    for G, s in zip(Gs, streams):
        with torch.cuda.stream(s):
            got.append(orthogonalize(G))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = [torch.zeros_like(G) for G in Gs]
    graphs, outs = [], []
    for x in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(orthogonalize(x))
        graphs.append(g)
    for round_ in range(4):
        for i in (0, 1):
            static[i].copy_(Gs[(i + round_) % 2])
        for g in graphs:
            g.replay()
        eager = orthogonalize(Gs[0])
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0])
        for i in (0, 1):
            assert torch.equal(outs[i], want[(i + round_) % 2])


@pytest.mark.gpu
def test_beside_the_estimators():
    """The handle's stream binding survives a call on another stream: the estimator's results stay."""
    from gaussian_process_amd import RBF, GaussianProcessRegression, orthogonalize
    rng = np.random.default_rng(0)
    X, y = rng.standard_normal((300, 2)), rng.standard_normal(300)

    def lml(between):
        gp = GaussianProcessRegression(cov=RBF(sigma=1.0, beta=0.5), sigma=0.1)
        gp.fit(X, y)
        if between:
            with torch.cuda.stream(torch.cuda.Stream()):
                orthogonalize(make((100, 100), "f64"))
        return gp.log_marginal_likelihood()

    assert lml(False) == lml(True)

"""The gated delta rule (chunked, backward, single tokens) against its recurrence in 64 bits.

Tolerances, relative in the 2-norm.  Sums run in fp32 over at most 128 + 64 terms a product (rounding grows like the
root of that: 14 x 2^-24), four products a chunk, and a decayed state carries the errors of the last few chunks: 14 * 2^-24 * 4 *
3 = 1e-5.  A result in fp16 or bf16 adds its own half step (2^-11, 2^-8).  d_g is a sum of differences of terms of up to ten
times its size: 1e-4."""
import numpy as np
import pytest
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
SUM = 1e-5


def rel(a, b):
    a = a.double().cpu().numpy() if isinstance(a, torch.Tensor) else a
    return np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-30)


def oracle(q, k, v, g, beta, state, offsets=None, scale=None, d_o=None, d_final=None):
    """o, final states and, with d_o, the gradients; token by token in 64 bits, gradients by the reversed recurrence."""
    q, k, v, g, beta, state = (np.asarray(x.double().cpu()) for x in (q, k, v, g, beta, state))
    B, T, Hk, dk = q.shape
    Hv, dv = v.shape[2:]
    r = Hv // Hk
    scale = dk ** -0.5 if scale is None else scale
    spans = [(b, 0, T) for b in range(B)] if offsets is None else [(0, offsets[i], offsets[i + 1]) for i in range(len(offsets) - 1)]
    o, final = np.zeros(v.shape), state.copy()
    back = d_o is not None
    if back:
        d_o, d_final = np.asarray(d_o.double().cpu()), np.asarray(d_final.double().cpu())
        dq, dk_, dv_, dg, db, ds = (np.zeros(x.shape) for x in (q, k, v, g, beta, state))
    for s, (b, t0, t1) in enumerate(spans):
        for h in range(Hv):
            S, kept = state[s, h], []
            for t in range(t0, t1):
                a = np.exp(g[b, t, h])
                bar = a * S
                e = v[b, t, h] - bar.T @ k[b, t, h // r]
                new = bar + beta[b, t, h] * np.outer(k[b, t, h // r], e)
                o[b, t, h] = scale * new.T @ q[b, t, h // r]
                kept.append((a, S, bar, e, new))
                S = new
            final[s, h] = S
            if not back:
                continue
            D = d_final[s, h]
            for t in reversed(range(t0, t1)):
                a, S, bar, e, new = kept[t - t0]
                qq, kk, w = q[b, t, h // r], k[b, t, h // r], beta[b, t, h]
                dq[b, t, h // r] += scale * new @ d_o[b, t, h]
                D = D + scale * np.outer(qq, d_o[b, t, h])
                db[b, t, h] = kk @ D @ e
                de = w * D.T @ kk
                dv_[b, t, h] = de
                dk_[b, t, h // r] += w * D @ e - bar @ de
                D = D - np.outer(kk, de)
                dg[b, t, h] = a * (D * S).sum()
                D = a * D
            ds[s, h] = D
    return (o, final, dq, dk_, dv_, dg, db, ds) if back else (o, final)


def inputs(B, T, Hk, Hv, dk, dv, kind="f32", seqs=None, seed=0, slow=False):
    rng = np.random.default_rng(seed)
    t = TYPES[kind]

    def unit(*shape):
        x = rng.standard_normal(shape) + 0.3
        return x / np.linalg.norm(x, axis=-1, keepdims=True)

    mk = lambda x, ty: torch.tensor(x).to(ty).cuda()  # noqa: E731
    g = -np.exp(rng.uniform(-5, -3 if slow else 0.5, (B, T, Hv)))
    return dict(q=mk(unit(B, T, Hk, dk), t), k=mk(unit(B, T, Hk, dk), t), v=mk(rng.standard_normal((B, T, Hv, dv)), t),
                g=mk(g, torch.float32), beta=mk(rng.uniform(0, 1.2, (B, T, Hv)), torch.float32),
                state=mk(0.5 * rng.standard_normal((seqs or B, Hv, dk, dv)), torch.float32))


def args(x):
    return [x[n] for n in ("q", "k", "v", "g", "beta")]


def cu(offsets):
    return torch.tensor(offsets, dtype=torch.int32, device="cuda")


def check(got, want, kind, names=("o", "final", "d_q", "d_k", "d_v", "d_g", "d_beta", "d_state")):
    for name, a, b in zip(names, got, want):
        typed = name in ("o", "d_q", "d_k", "d_v")
        tol = (1e-4 if name == "d_g" else SUM) + (HALF[kind] if typed else 0)
        assert tuple(a.shape) == b.shape
        assert rel(a, b) < tol, (name, rel(a, b), tol)


def both(x, kind, offsets=None, seed=5, scale=None):
    """forward, saving forward and backward against the oracle"""
    from gaussian_process_amd import gated_delta_rule, gated_delta_rule_backward
    rng = np.random.default_rng(seed)
    d_o = torch.tensor(rng.standard_normal(x["v"].shape)).to(x["v"].dtype).cuda()
    d_f = torch.tensor(0.3 * rng.standard_normal(x["state"].shape)).float().cuda()
    c = None if offsets is None else cu(offsets)
    want = oracle(*args(x), x["state"], offsets, scale, d_o, d_f)
    o, f = gated_delta_rule(*args(x), initial_state=x["state"], cu_seqlens=c, scale=scale)
    check((o, f), want, kind)
    o2, f2, saved = gated_delta_rule(*args(x), initial_state=x["state"], cu_seqlens=c, scale=scale, save_for_backward=True)
    check((o2, f2, *gated_delta_rule_backward(saved, d_o, d_f)), want, kind)
    return want


# ---- refusals (no GPU) --------------------------------------------------------------------------------------------
def host(B=2, T=3, Hk=1, Hv=2, dk=4, dv=5, t=torch.float32):
    return [torch.zeros(B, T, Hk, dk, dtype=t), torch.zeros(B, T, Hk, dk, dtype=t), torch.zeros(B, T, Hv, dv, dtype=t),
            torch.zeros(B, T, Hv), torch.zeros(B, T, Hv)]


def test_refusals():
    from gaussian_process_amd import _lib, gated_delta_rule, gated_delta_rule_backward, gated_delta_rule_step
    with pytest.raises(_lib.GpxError):
        gated_delta_rule(*host())
    with pytest.raises(TypeError):
        gated_delta_rule(*host(t=torch.float64))
    with pytest.raises(TypeError):
        gated_delta_rule(*host()[:2], host(t=torch.float16)[2], *host()[3:])
    with pytest.raises(TypeError):
        gated_delta_rule(*host()[:3], host()[3].double(), host()[4])
    with pytest.raises(TypeError):
        gated_delta_rule(*host()[:4], None)
    for bad in (dict(dk=129), dict(dk=0), dict(dv=0), dict(dv=1025), dict(Hk=2, Hv=3), dict(Hk=0, Hv=0)):
        with pytest.raises(ValueError):
            gated_delta_rule(*host(**bad))
    x = host()
    for i, shape in ((0, (2, 3, 1, 5)), (1, (2, 4, 1, 4)), (2, (2, 3, 2)), (3, (2, 3, 1)), (4, (2, 3, 2, 1))):
        y = list(x)
        y[i] = torch.zeros(shape)
        with pytest.raises(ValueError):
            gated_delta_rule(*y)
    with pytest.raises(ValueError):
        gated_delta_rule(*x, initial_state=torch.zeros(2, 2, 5, 4))
    with pytest.raises(ValueError):
        gated_delta_rule(*x, initial_state=torch.zeros(2, 2, 4, 5, dtype=torch.float64))
    with pytest.raises(ValueError):   # packed sequences and a batch
        gated_delta_rule(*x, cu_seqlens=torch.zeros(3, dtype=torch.int32))
    for c in (torch.zeros(3), torch.zeros(1, dtype=torch.int32), torch.zeros(3, 1, dtype=torch.int32)):
        with pytest.raises(ValueError):
            gated_delta_rule(*host(B=1), cu_seqlens=c)
    with pytest.raises(TypeError):
        gated_delta_rule_backward(None, x[2])
    row = [t[:, 0] for t in x]
    st = torch.zeros(2, 2, 4, 5)
    with pytest.raises(_lib.GpxError):
        gated_delta_rule_step(*row, st)
    for kw in (dict(state=torch.zeros(3, 2, 4, 5)), dict(state=st, slots=torch.zeros(2)), dict(state=st.mT.contiguous().mT),
               dict(state=st, slots=torch.zeros(3, dtype=torch.int32)), dict(state=st, state_out=torch.zeros(3, 2, 4, 5)),
               dict(state=st, state_out=torch.zeros(2, 2, 4, 5).half())):
        with pytest.raises(ValueError):
            gated_delta_rule_step(*row, **kw)
    pool = torch.zeros(3, 2, 4, 5)
    with pytest.raises(ValueError):
        gated_delta_rule_step(*row, pool[:2], state_out=pool[1:])


def desc(**kw):
    from gaussian_process_amd import _lib
    base = dict(dtype=3, batch=2, tokens=100, sequences=0, key_heads=2, value_heads=4, dk=64, dv=40, scale=1.0)
    base.update(kw)
    d = _lib.Delta()
    for name, value in base.items():
        setattr(d, name, value)
    for name in ("q", "k", "v", "g", "beta"):
        setattr(d, name, 256)
    return d


def test_work_bytes():
    import ctypes as C
    from gaussian_process_amd import _lib
    lib = _lib.load()
    w = lambda use, **kw: lib.gpx_delta_work_bytes(C.byref(desc(**kw)), use)  # noqa: E731
    heads, kheads = 2 * 2 * 4, 2 * 2 * 2   # rows, chunks, heads; dv rounded up to 64, dk to 64
    square = 64 * 64                       # elements of a fragment-wise C x C or dk x C matrix; K and Q take two
    both_ = heads * (64 * 8 + 6 * 64 * 4) + kheads * 3 * square * 2
    work = kheads * 2 * square * 2 + heads * 5 * square * 2
    assert w(0) == both_ + work and w(3) == work
    assert w(1) == both_ + kheads * square * 2 + heads * (6 * square * 2 + (64 + 64) * 64 * 4)
    assert w(2) == heads * (64 + 64) * 64 * 4 + 2 * heads * square * 4   # value heads apart: their parts of d_q and d_k
    assert w(2, batch=40) == 20 * heads * (64 + 64) * 64 * 4 and w(2, key_heads=4) == heads * (64 + 64) * 64 * 4
    assert w(0, tokens=16) == 0                                   # the recurrence needs none
    assert w(0, tokens=16, batch=1, sequences=5, offsets=256) == 256
    assert w(4) == 0 and w(0, dk=129) == 0 and w(0, dtype=0) == 0 and w(0, value_heads=3) == 0
    assert w(1, batch=1, sequences=5, offsets=256) == 256 + w(1) * 6 // 4
    assert w(0, batch=1, sequences=5) == 0                       # no offsets
    assert w(1, batch=1 << 24, tokens=1 << 30) == 0              # beyond the grid
    big = dict(batch=1 << 20, key_heads=16, value_heads=16, dv=128)
    assert w(0, tokens=64, **big) == 0 and w(1, tokens=1, **big) == 0 and w(0, tokens=64, **{**big, "batch": 1 << 15}) > 0


# ---- GPU ----------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 63, 64, 65, 130])
@pytest.mark.parametrize("kind", list(TYPES))
def test_lengths(T, kind):
    both(inputs(2, T, 1, 2, 64, 32, kind, seed=T), kind)


@pytest.mark.gpu
@pytest.mark.parametrize("Hk,Hv,dk,dv", [(1, 1, 1, 1), (1, 3, 16, 16), (2, 4, 100, 33), (2, 2, 65, 130), (1, 2, 128, 128),
                                         (3, 3, 128, 7), (1, 1, 7, 200)])
@pytest.mark.parametrize("kind", list(TYPES))
def test_heads_and_sizes(Hk, Hv, dk, dv, kind):
    both(inputs(2, 90, Hk, Hv, dk, dv, kind, seed=dk), kind, scale=0.7)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("offsets", [[0, 150], [0, 0, 1, 1, 65, 129, 150, 150], [0, 64, 128, 150], [7, 7, 71, 140], [0, 0], [150, 150, 150]])
def test_ragged(offsets, kind):
    n = len(offsets) - 1
    x = inputs(1, 150, 2, 4, 48, 40, kind, seqs=n, seed=n)
    both(x, kind, offsets)


@pytest.mark.gpu
def test_short_ragged():
    for T, offsets in ((9, [0, 0, 3, 4, 9]), (1, [0, 1, 1])):
        both(inputs(1, T, 1, 2, 32, 20, "f32", seqs=len(offsets) - 1), "f32", offsets)


@pytest.mark.gpu
@pytest.mark.parametrize("dk,dv", [(128, 128), (40, 100)])
def test_more_workgroups_than_compute_units(dk, dv):
    both(inputs(3, 150, 7, 14, dk, dv, "bf16", seed=dk), "bf16")


@pytest.mark.gpu
def test_many_sequences():
    """More sequences than one wave's lanes, most of them short or empty, a few long ones last."""
    rng = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 12, (150,), generator=rng).tolist() + [300, 65, 500]
    offsets = [0]
    for n in lens:
        offsets.append(offsets[-1] + n)
    both(inputs(1, offsets[-1], 1, 2, 32, 24, "f32", seqs=len(lens), seed=9), "f32", offsets)


@pytest.mark.gpu
def test_bad_offsets_stay_inside():
    """Values outside the tokens are clamped, decreasing ones read as the one before."""
    from gaussian_process_amd import gated_delta_rule, gated_delta_rule_backward
    x = inputs(1, 150, 1, 2, 64, 32, "bf16", seqs=4)
    d_o = torch.ones_like(x["v"])
    good, bad = [0, 70, 70, 150, 150], [-5, 70, 20, 1 << 30, -(1 << 31)]
    outs = []
    for c in (good, bad):
        o, f, saved = gated_delta_rule(*args(x), initial_state=x["state"], cu_seqlens=cu(c), save_for_backward=True)
        outs.append((o, f, *gated_delta_rule_backward(saved, d_o)))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.gpu
def test_no_tokens_and_no_rows():
    from gaussian_process_amd import gated_delta_rule, gated_delta_rule_backward, gated_delta_rule_step
    x = inputs(2, 0, 1, 2, 16, 16)
    o, f, saved = gated_delta_rule(*args(x), initial_state=x["state"], save_for_backward=True)
    assert o.shape == (2, 0, 2, 16) and torch.equal(f, x["state"])
    d = torch.randn_like(f)
    grads = gated_delta_rule_backward(saved, torch.empty_like(x["v"]), d)
    assert torch.equal(grads[-1], d) and grads[0].shape == x["q"].shape
    x = inputs(1, 0, 1, 2, 16, 16, seqs=3)
    o, f = gated_delta_rule(*args(x), initial_state=x["state"], cu_seqlens=cu([0, 0, 0, 0]))
    assert torch.equal(f, x["state"])
    x = inputs(0, 5, 1, 2, 16, 16)
    o, f = gated_delta_rule(*args(x))
    assert o.shape == (0, 5, 2, 16) and f.shape == (0, 2, 16, 16)
    o, f = gated_delta_rule_step(*(t[:, 0] for t in args(x)), f)
    assert o.shape == (0, 2, 16)
    x = inputs(2, 1, 1, 2, 16, 16)
    o, f = gated_delta_rule_step(*(t[:, 0] for t in args(x)), x["state"][:0], slots=cu([0, -1]))
    assert (o == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_resets_padding_and_strong_decay(kind):
    """g = -inf forgets, beta = 0 with g = 0 changes nothing, decays that underflow and large ones stay finite."""
    x = inputs(2, 140, 1, 2, 64, 32, kind, seed=8)
    x["g"][0, 5, 0] = -float("inf")
    x["g"][:, 64] = -float("inf")
    x["g"][1, 100:, 1] = -float("inf")
    x["g"][0, 20:40, 1] = -150.0
    x["g"][1, 10:30] = 0
    x["beta"][1, 10:30] = 0
    x["beta"][0, 130:, 0] = 0
    x["beta"][0, 50:60, 1] = 2.0
    want = both(x, kind)
    assert all(np.isfinite(w).all() for w in want)


@pytest.mark.gpu
def test_nan_stays_in_its_sequence():
    from gaussian_process_amd import gated_delta_rule
    x = inputs(1, 200, 1, 2, 64, 32, "bf16", seqs=3)
    off = [0, 50, 120, 200]
    want = oracle(*args(x), x["state"], off)
    x["v"][0, 60, 0, 3] = float("nan")
    x["state"][1, 1] = float("inf")
    o, f = gated_delta_rule(*args(x), initial_state=x["state"], cu_seqlens=cu(off))
    for sl, s in ((slice(0, 50), 0), (slice(120, 200), 2)):
        assert rel(o[0, sl], want[0][0, sl]) < SUM + HALF["bf16"] and rel(f[s], want[1][s]) < SUM
    assert o[0, 60:120, 0, 3].isnan().all()


@pytest.mark.gpu
def test_no_state_given():
    from gaussian_process_amd import gated_delta_rule, gated_delta_rule_backward
    for T in (5, 100):
        x = inputs(2, T, 1, 2, 32, 32)
        zero = torch.zeros_like(x["state"])
        d_o = torch.randn_like(x["v"])
        want = oracle(*args(x), zero, d_o=d_o, d_final=zero)
        o, f, saved = gated_delta_rule(*args(x), save_for_backward=True)
        grads = gated_delta_rule_backward(saved, d_o)
        assert grads[-1] is None
        check((o, f, *grads[:-1]), want[:-1], "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_strides(kind):
    """Views: heads before tokens, every other token, a slice of a fused projection, an expanded and a transposed one."""
    from gaussian_process_amd import gated_delta_rule, gated_delta_rule_backward
    B, T, Hk, Hv, dk, dv = 2, 80, 2, 4, 40, 24
    x = inputs(B, T, Hk, Hv, dk, dv, kind)
    want = both(x, kind)
    y = dict(x)
    y["q"] = x["q"].transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.zeros(B, T, Hk, dk + 3, dtype=x["k"].dtype, device="cuda")
    wide[..., 1:dk + 1] = x["k"]
    y["k"] = wide[..., 1:dk + 1]
    twice = torch.zeros(B, 2 * T, Hv, dv, dtype=x["v"].dtype, device="cuda")
    twice[:, ::2] = x["v"]
    y["v"] = twice[:, ::2]
    y["g"] = x["g"].permute(2, 0, 1).contiguous().permute(1, 2, 0)
    y["beta"] = torch.stack([x["beta"], x["beta"]], -1)[..., 1]
    y["state"] = x["state"].mT.contiguous().mT
    d_o = torch.tensor(np.random.default_rng(5).standard_normal(x["v"].shape)).to(x["v"].dtype).cuda()
    rng = np.random.default_rng(5)
    rng.standard_normal(x["v"].shape)
    d_f = torch.tensor(0.3 * rng.standard_normal(x["state"].shape)).float().cuda()
    o, f, saved = gated_delta_rule(*args(y), initial_state=y["state"], save_for_backward=True)
    got = (o, f, *gated_delta_rule_backward(saved, d_o.mT.contiguous().mT, d_f.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)))
    check(got, want, kind)
    # the last dimension not dense; one token for all
    y["q"] = x["q"].mT.contiguous().mT
    y["k"] = x["k"][:, :1].expand(-1, T, -1, -1)
    z = dict(x, k=y["k"].contiguous())
    check(gated_delta_rule(y["q"], y["k"], *args(x)[2:], initial_state=x["state"]), oracle(*args(z), x["state"]), kind)


@pytest.mark.gpu
def test_gradients_by_differences():
    """Central differences of the 64-bit recurrence in random directions, so that the oracle's own gradients are checked."""
    x = inputs(1, 70, 1, 2, 16, 12)
    rng = np.random.default_rng(1)
    d_o, d_f = torch.randn_like(x["v"]), torch.randn_like(x["state"])
    want = both(x, "f32")
    got = oracle(*args(x), x["state"], d_o=d_o, d_final=d_f)[2:]
    assert len(want) == 8

    def loss(y):
        o, f = oracle(*args(y), y["state"])
        return (o * d_o.double().cpu().numpy()).sum() + (f * d_f.double().cpu().numpy()).sum()

    for name, grad in zip(("q", "k", "v", "g", "beta", "state"), got):
        way = rng.standard_normal(grad.shape)
        h = 1e-5
        up, down = ({**x, name: x[name].double() + s * h * torch.tensor(way).cuda()} for s in (1, -1))
        slope = (loss(up) - loss(down)) / (2 * h)
        assert abs(slope - (grad * way).sum()) < 1e-6 * np.linalg.norm(grad) * np.linalg.norm(way)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("B,Hk,Hv,dk,dv", [(1, 1, 1, 1, 1), (3, 2, 4, 64, 64), (2, 1, 3, 100, 33), (5, 2, 2, 128, 128), (2, 1, 2, 20, 130)])
def test_step(B, Hk, Hv, dk, dv, kind):
    from gaussian_process_amd import gated_delta_rule_step
    x = inputs(B, 4, Hk, Hv, dk, dv, kind)
    want_o, want_f = oracle(*args(x), x["state"])
    state = x["state"].clone()
    for t in range(4):
        o, s = gated_delta_rule_step(*(y[:, t] for y in args(x)), state)
        assert s is state and rel(o, want_o[:, t]) < SUM + HALF[kind]
    assert rel(state, want_f) < SUM
    other = torch.full_like(state, 7.0)
    o1, s = gated_delta_rule_step(*(y[:, 0] for y in args(x)), x["state"], state_out=other)
    assert s is other and rel(o1, want_o[:, 0]) < SUM + HALF[kind]


@pytest.mark.gpu
def test_step_slots():
    """Rows name states of a pool: padding, out of range, a slot twice and three times (far apart too), states left alone."""
    from gaussian_process_amd import gated_delta_rule_step
    B, n = 150, 9
    x = inputs(B, 1, 1, 2, 64, 40, "f32")
    pool = torch.randn(n, 2, 64, 40, device="cuda")
    rows = [-1] * B
    for r, s in ((0, 3), (1, 8), (2, n), (70, 3), (71, 0), (130, 3), (149, 8), (20, 1 << 30), (21, -(1 << 31)), (140, 5)):
        rows[r] = s
    slots = cu(rows)
    want_pool, want_o = pool.double().cpu().numpy(), np.zeros((B, 2, 40))
    for r, s in enumerate(rows):
        if 0 <= s < n:
            o, f = oracle(*(y[r:r + 1] for y in args(x)), torch.tensor(want_pool[s:s + 1]))
            want_o[r], want_pool[s] = o[0, 0], f[0]
    other = pool.clone()
    o, s = gated_delta_rule_step(*(y[:, 0] for y in args(x)), pool, slots=slots, state_out=other)
    assert rel(o, want_o) < SUM and rel(other, want_pool) < SUM
    untouched = [i for i in range(n) if i not in rows]
    assert torch.equal(other[untouched], pool[untouched])
    assert (o[[r for r in range(B) if not 0 <= rows[r] < n]] == 0).all()
    again = pool.clone()
    gated_delta_rule_step(*(y[:, 0] for y in args(x)), again, slots=slots)
    assert torch.equal(again, other)


@pytest.mark.gpu
def test_chunks_and_recurrence_agree():
    """The same sequence in one call, in pieces through the state, and token by token."""
    from gaussian_process_amd import gated_delta_rule, gated_delta_rule_step
    x = inputs(2, 150, 1, 2, 64, 64, "f32", slow=True)
    whole, f = gated_delta_rule(*args(x), initial_state=x["state"])
    s, parts = x["state"], []
    for a, b in ((0, 70), (70, 71), (71, 80), (80, 150)):
        o, s = gated_delta_rule(*(y[:, a:b] for y in args(x)), initial_state=s)
        parts.append(o)
    want = oracle(*args(x), x["state"])
    check((whole, f), want, "f32")
    check((torch.cat(parts, 1), s), want, "f32")
    s, parts = x["state"].clone(), []
    for t in range(150):
        parts.append(gated_delta_rule_step(*(y[:, t] for y in args(x)), s)[0])
    check((torch.stack(parts, 1), s), want, "f32")


@pytest.mark.gpu
def test_saved_is_only_read_and_guarded():
    from gaussian_process_amd import gated_delta_rule, gated_delta_rule_backward
    x = inputs(2, 100, 1, 2, 64, 64, "bf16")
    o, f, saved = gated_delta_rule(*args(x), initial_state=x["state"], save_for_backward=True)
    d1, d2 = torch.randn_like(o), torch.randn_like(o)
    first = gated_delta_rule_backward(saved, d1)
    gated_delta_rule_backward(saved, d2)
    assert all(torch.equal(a, b) for a, b in zip(first, gated_delta_rule_backward(saved, d1)))
    with pytest.raises(ValueError):
        gated_delta_rule_backward(saved, d1.float())
    with pytest.raises(ValueError):
        gated_delta_rule_backward(saved, d1, f[:1])
    x["k"].mul_(2)
    with pytest.raises(RuntimeError):
        gated_delta_rule_backward(saved, d1)


@pytest.mark.gpu
def test_saved_notices_writes_of_this_package():
    from gaussian_process_amd import gated_delta_rule, gated_delta_rule_backward, gated_delta_rule_step, orthogonalize
    x = inputs(1, 70, 1, 1, 16, 16, "f32")
    o, f, saved = gated_delta_rule(*args(x), save_for_backward=True)
    orthogonalize(x["v"], out=x["v"])
    with pytest.raises(RuntimeError):
        gated_delta_rule_backward(saved, torch.ones_like(o))
    before = f._version
    gated_delta_rule_step(*(t[:, 0] for t in args(x)), f)
    assert f._version > before


@pytest.mark.gpu
def test_backward_on_another_stream():
    from gaussian_process_amd import gated_delta_rule, gated_delta_rule_backward
    x = inputs(2, 200, 2, 4, 64, 64, "bf16")
    d_o = torch.randn_like(x["v"])
    want = gated_delta_rule_backward(gated_delta_rule(*args(x), save_for_backward=True)[2], d_o)
    side = torch.cuda.Stream()
    saved = gated_delta_rule(*args(x), save_for_backward=True)[2]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gated_delta_rule_backward(saved, d_o)
    del saved
    torch.full((1 << 24,), float("nan"), device="cuda")   # where the saved values were, if they were given back too early
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got) if a is not None)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_streams_and_graphs(kind):
    """Forward and backward at once on two streams; captured, replayed with other inputs and eager work between."""
    from gaussian_process_amd import gated_delta_rule, gated_delta_rule_backward, gated_delta_rule_step
    off = [0, 30, 30, 140]
    xs = [inputs(1, 140, 1, 2, 64, 40, kind, seqs=3, seed=i) for i in (1, 2)]
    d_o = torch.randn(1, 140, 2, 40, device="cuda").to(TYPES[kind])
    c = cu(off)

    def go(x):
        o, f, saved = gated_delta_rule(*args(x), initial_state=x["state"], cu_seqlens=c, save_for_backward=True)
        grads = gated_delta_rule_backward(saved, d_o, f)
        state = torch.empty_like(f)
        one, _ = gated_delta_rule_step(*(y[0, :3] for y in args(x)), x["state"], state_out=state)
        return (o, f, *grads, one, state, *gated_delta_rule(*args(x), cu_seqlens=c))

    want = [go(x) for x in xs]
    torch.cuda.synchronize()
    got = []
    for x in xs:
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(go(x))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    static = [{n: t.clone() for n, t in xs[0].items()} for _ in range(2)]
    graphs, outs = [], []
    for x in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(go(x))
        graphs.append(g)
    for turn in range(4):
        for i in (0, 1):
            for n in static[i]:
                static[i][n].copy_(xs[(i + turn) % 2][n])
        for g in graphs:
            g.replay()
        eager = go(xs[0])
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(eager, want[0]))
        for i in (0, 1):
            assert all(torch.equal(p, q) for p, q in zip(outs[i], want[(i + turn) % 2]))


@pytest.mark.gpu
def test_train_and_serve():
    """As they are used together: keys, queries and values are learned projections of a stream; the gradients through the
    delta rule and the projections, checked against 64 bits; the projections moved by orthogonalised updates; then the
    stream served token by token with the moved weights gives what one call over all of it gives."""
    from gaussian_process_amd import gated_delta_rule, gated_delta_rule_backward, gated_delta_rule_step, orthogonalize
    rng = np.random.default_rng(3)
    B, T, D, Hk, Hv, dk, dv = 2, 90, 48, 1, 2, 32, 24
    h = torch.tensor(rng.standard_normal((B, T, D))).float().cuda()
    target = torch.tensor(rng.standard_normal((B, T, Hv, dv))).float().cuda()
    W = {n: torch.tensor(rng.standard_normal((D, w)) * D ** -0.5).float().cuda() for n, w in (("q", Hk * dk), ("k", Hk * dk), ("v", Hv * dv))}
    g = torch.full((B, T, Hv), -0.02, device="cuda")
    beta = torch.full((B, T, Hv), 0.1, device="cuda")

    def project(W, h):
        return [(h @ W[n] * (0.3 if n == "k" else 1)).view(*h.shape[:-1], Hv if n == "v" else Hk, -1) for n in ("q", "k", "v")]

    for _ in range(2):
        q, k, v = project(W, h)
        o, f, saved = gated_delta_rule(q, k, v, g, beta, save_for_backward=True)
        d_o = o - target
        grads = gated_delta_rule_backward(saved, d_o)[:3]
        zero = torch.zeros(B, Hv, dk, dv)
        want = oracle(q, k, v, g, beta, zero, d_o=d_o, d_final=zero)
        check((o, f, *grads), want, "f32")
        for n, d, c in zip(("q", "k", "v"), grads, (1, 0.3, 1)):
            dW = c * h.reshape(-1, D).T @ d.reshape(B * T, -1)
            before = W[n].clone()
            orthogonalize(dW, alpha=-0.05, beta=0.99, base=W[n], out=W[n])
            s = np.linalg.svd(((0.99 * before - W[n]) / 0.05).double().cpu().numpy(), compute_uv=False)
            assert s.max() < 1.25
    q, k, v = project(W, h)
    o, f = gated_delta_rule(q, k, v, g, beta)
    state = torch.zeros(B, Hv, dk, dv, device="cuda")
    served = torch.stack([gated_delta_rule_step(*(y[:, t] for y in (q, k, v, g, beta)), state)[0] for t in range(T)], 1)
    assert rel(served, o.double().cpu().numpy()) < 2 * SUM and rel(state, f.double().cpu().numpy()) < 2 * SUM

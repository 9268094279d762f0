"""The delta rule where chunks are many: the variants that are chosen by the number of chunks times value heads (256 and 512), with shared
key heads, whose results small cases never see; against the recurrence in 64 bits, with the tolerances of test_delta_rule.py, d_g head by head."""
import numpy as np
import pytest
import torch

from test_delta_rule import TYPES, args, check, cu, inputs


def oracle(x, offsets, scale, d_o, d_final):
    """As test_delta_rule.py's, with all sequences and heads at once: an ended sequence's g is 0 and its beta 0."""
    q, k, v, g, beta, state = (x[n].double().cpu().numpy() for n in ("q", "k", "v", "g", "beta", "state"))
    d_o, d_final = d_o.double().cpu().numpy(), d_final.double().cpu().numpy()
    B, T, Hv = g.shape
    group = Hv // q.shape[2]
    spans = [(b, 0, T) for b in range(B)] if offsets is None else [(0, a, b) for a, b in zip(offsets, offsets[1:])]
    longest = max(b - a for _, a, b in spans)

    def lay(y):   # (longest, sequences, heads, ...)
        out = np.zeros((longest, len(spans)) + y.shape[2:])
        for s, (b, t0, t1) in enumerate(spans):
            out[:t1 - t0, s] = y[b, t0:t1]
        return out

    def back(y, like):
        out = np.zeros(like.shape)
        for s, (b, t0, t1) in enumerate(spans):
            out[b, t0:t1] = y[:t1 - t0, s]
        return out

    wide = lambda y: np.repeat(y, group, 2)   # noqa: E731
    Q, K, V, A, W, D = lay(wide(q)), lay(wide(k)), lay(v), np.exp(lay(g)), lay(beta), lay(d_o)
    S, kept, O = state, [], np.zeros_like(V)
    for t in range(longest):
        bar = A[t][..., None, None] * S
        e = V[t] - np.einsum("shk,shkv->shv", K[t], bar)
        new = bar + W[t][..., None, None] * K[t][..., :, None] * e[..., None, :]
        O[t] = scale * np.einsum("shk,shkv->shv", Q[t], new)
        kept.append((S, bar, e, new))
        S = new
    final, dS = S, d_final
    dq, dk, dv, dg, db = (np.zeros_like(y) for y in (Q, K, V, A, W))
    for t in reversed(range(longest)):
        S, bar, e, new = kept.pop()
        dq[t] = scale * np.einsum("shkv,shv->shk", new, D[t])
        dS = dS + scale * Q[t][..., :, None] * D[t][..., None, :]
        down = np.einsum("shk,shkv->shv", K[t], dS)
        db[t] = (down * e).sum(-1)
        dv[t] = W[t][..., None] * down
        dk[t] = W[t][..., None] * np.einsum("shkv,shv->shk", dS, e) - np.einsum("shkv,shv->shk", bar, dv[t])
        dS = dS - K[t][..., :, None] * dv[t][..., None, :]
        dg[t] = A[t] * (dS * S).sum((-2, -1))
        dS = A[t][..., None, None] * dS
    shared = lambda y: y.reshape(y.shape[:2] + (-1, group) + y.shape[3:]).sum(3)   # noqa: E731
    return (back(O, v), final, back(shared(dq), q), back(shared(dk), k), back(dv, v), back(dg, g), back(db, beta), dS)


def slots(offsets, B, T):
    return B * ((T + 63) // 64) if offsets is None else T // 64 + len(offsets) - 1


def run(kind, B, T, Hk, Hv, dk, dv, offsets, seed):
    from gaussian_process_amd import gated_delta_rule, gated_delta_rule_backward
    x = inputs(B, T, Hk, Hv, dk, dv, kind, seqs=None if offsets is None else len(offsets) - 1, seed=seed)
    rng = np.random.default_rng(seed)
    d_o = torch.tensor(rng.standard_normal(x["v"].shape)).to(TYPES[kind]).cuda()
    d_f = torch.tensor(0.3 * rng.standard_normal(x["state"].shape)).float().cuda()
    c = None if offsets is None else cu(offsets)
    want = oracle(x, offsets, 0.7, d_o, d_f)
    check(gated_delta_rule(*args(x), initial_state=x["state"], cu_seqlens=c, scale=0.7), want, kind)
    o, f, saved = gated_delta_rule(*args(x), initial_state=x["state"], cu_seqlens=c, scale=0.7, save_for_backward=True)
    got = (o, f, *gated_delta_rule_backward(saved, d_o, d_f))
    check(got, want, kind)
    for h in range(Hv):
        a, b = got[5][..., h].double().cpu().numpy(), want[5][..., h]
        assert np.linalg.norm(a - b) < 1e-4 * np.linalg.norm(b)


def ragged(T, n, seed):
    cuts = np.random.default_rng(seed).integers(0, T + 1, n - 1)
    return [0, *sorted(cuts.tolist()), T]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("Hk,Hv", [(4, 8), (2, 6), (5, 5)])
@pytest.mark.parametrize("dk,dv", [(64, 32), (100, 20), (128, 33)])
@pytest.mark.parametrize("least", [257, 513])
def test_batches(kind, Hk, Hv, dk, dv, least):
    B = -(-least // (2 * Hv))
    assert (256 if least == 257 else 512) < slots(None, B, 70) * Hv <= (512 if least == 257 else 600)
    run(kind, B, 70, Hk, Hv, dk, dv, None, seed=dk + Hv)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("Hk,Hv,dk,dv", [(4, 8, 64, 48), (3, 9, 100, 16), (2, 4, 128, 64), (6, 6, 128, 24)])
@pytest.mark.parametrize("least", [257, 513])
def test_packed(kind, Hk, Hv, dk, dv, least):
    n = -(-least // Hv)   # slots: two in three a sequence of its own
    offsets = ragged(64 * (n // 3), n - n // 3, seed=n)
    T = offsets[-1]
    assert (256 if least == 257 else 512) < slots(offsets, 1, T) * Hv <= (512 if least == 257 else 600)
    run(kind, 1, T, Hk, Hv, dk, dv, offsets, seed=dk)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_unaligned_rows(kind):
    """Sizes that leave no 16-byte rows of d_q, d_k and d_v."""
    run(kind, 22, 70, 4, 12, 37, 21, None, seed=5)

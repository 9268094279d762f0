"""Cases of the operators that learn and carry a matrix: the gated delta rule (chunked forward, forward with
backward, single tokens) and the orthogonalisation of an update by Newton-Schulz products.

Conventions: q, k are (B, T, Hk, dk), v and o (B, T, Hv, dv), Hv a multiple of Hk; g (log decay, <= 0) and beta
(B, T, Hv) in float32; states (sequences, Hv, dk, dv) in float32.  Ragged batches are packed as B = 1 with offsets.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f64": 8, "f32": 4, "f16": 2, "bf16": 2}
STEPS = 5
COEF = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
CHUNK = 64


def listed():
    return [
        # the projection of one head of a small model: launch latency counts
        dict(name="orth_128x512_f32", op="orth", batch=1, n=128, m=512, type="f32", base=False),
        # one square projection of a small model, gradients in half width
        dict(name="orth_1024x1024_bf16", op="orth", batch=1, n=1024, m=1024, type="bf16", base=False),
        # the largest: a square projection of a large model
        dict(name="orth_4096x4096_bf16", op="orth", batch=1, n=4096, m=4096, type="bf16", base=False),
        # a wide feed-forward weight with float32 master weights, updated in the same call: W <- 0.99 W - 0.02 O
        dict(name="orth_2048x8192_f32_update", op="orth", batch=1, n=2048, m=8192, type="f32", base=True),
        # a stack of tall ragged matrices (experts), transposed inside
        dict(name="orth_8x1300x777_f16", op="orth", batch=8, n=1300, m=777, type="f16", base=False),
        # the framework's own type
        dict(name="orth_1024x2048_f64", op="orth", batch=1, n=1024, m=2048, type="f64", base=False),
        # one long document read in
        dict(name="delta_fwd_8192_bf16", op="fwd", B=1, T=8192, Hk=16, Hv=16, dk=128, dv=128, type="bf16", seqs=0),
        # a packed batch of ragged prompts, key heads shared by two value heads
        dict(name="delta_fwd_ragged_f16", op="fwd", B=1, T=5003, Hk=4, Hv=8, dk=128, dv=128, type="f16", seqs=9),
        # a training step of one layer
        dict(name="delta_train_2x4096_bf16", op="train", B=2, T=4096, Hk=16, Hv=16, dk=128, dv=128, type="bf16", seqs=0),
        # a small odd model in float32, shared key heads, ragged sequences
        dict(name="delta_train_ragged_f32", op="train", B=1, T=700, Hk=2, Hv=4, dk=96, dv=65, type="f32", seqs=4),
        # a serving step of a full batch: every sequence gets one token
        dict(name="delta_step_64_bf16", op="step", B=64, Hk=16, Hv=32, dk=128, dv=128, type="bf16"),
        # one user
        dict(name="delta_step_1_bf16", op="step", B=1, Hk=8, Hv=8, dk=64, dv=64, type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["orth", "orth", "fwd", "train", "step"])
    if op == "orth":
        kind = rng.choice(["f32", "f32", "f16", "bf16", "bf16", "f64"])
        top = 1400 if kind == "f64" else 4096
        while True:
            n, m, batch = _log(rng, 16, top), _log(rng, 16, 2 * top), rng.choice([1, 1, 2, 5])
            small, large = min(n, m), max(n, m)
            if batch * small * small * (small + 3 * large) <= (4 if kind == "f64" else 270) * 1e9:
                return dict(op=op, batch=batch, n=n, m=m, type=kind, base=rng.random() < 0.3)
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    group = rng.choice([1, 1, 2, 3])
    dk, dv = rng.choice([64, 128, 128, rng.randint(16, 128)]), rng.choice([64, 128, 128, rng.randint(16, 160)])
    if op == "step":
        Hk = _log(rng, 1, 16)
        return dict(op=op, B=_log(rng, 1, 128), Hk=Hk, Hv=Hk * group, dk=dk, dv=dv, type=kind)
    seqs = rng.choice([0, _log(rng, 1, 24)])
    Hk = _log(rng, 1, 8)
    B = 1 if seqs else rng.choice([1, 1, 2, 4])
    T = _log(rng, 1, (8192 if op == "fwd" else 4096) // B)
    return dict(op=op, B=B, T=T, Hk=Hk, Hv=Hk * group, dk=dk, dv=dv, type=kind, seqs=seqs)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _offsets(case, seed):
    """Ends of the packed sequences: cuts at random places, so some are long and some empty; None for a plain batch."""
    if not case["seqs"]:
        return None
    r = torch.Generator().manual_seed(seed + 1)
    cuts = torch.sort(torch.randint(0, case["T"] + 1, (case["seqs"] - 1,), generator=r)).values.tolist()
    return [0] + cuts + [case["T"]]


def prepare(case, seed):
    g_ = _gen(seed)
    t = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, generator=g_, device=DEV)

    if case["op"] == "orth":
        b, n, m = case["batch"], case["n"], case["m"]
        # gradients of weights: a few strong directions over noise
        r = min(8, n, m)
        G = normal(b, n, m) + (normal(b, n, r) * torch.linspace(4, 0.5, r, device=DEV)) @ normal(b, r, m)
        base = normal(b, n, m) * m ** -0.5 if case["base"] else None
        if b == 1:
            G, base = G[0], base[0] if base is not None else None
        return dict(case=case, G=(G * 1e-3).to(t), base=base.to(t) if base is not None else None)
    B, T = case["B"], case.get("T", 1)
    Hk, Hv, dk, dv = case["Hk"], case["Hv"], case["dk"], case["dv"]

    def unit(*shape):  # keys and queries of unit length, with a common direction: neighbours are correlated
        x = normal(*shape) + 0.5 * normal(shape[0], 1, *shape[2:])
        return x / x.norm(dim=-1, keepdim=True)

    s = dict(case=case, q=unit(B, T, Hk, dk).to(t), k=unit(B, T, Hk, dk).to(t), v=normal(B, T, Hv, dv).to(t),
             beta=torch.sigmoid(normal(B, T, Hv)),
             # decay rates from slow heads (0.001 a token) to fast ones (1 a token and more)
             g=-torch.nn.functional.softplus(normal(B, T, Hv)) * torch.logspace(-3, 0, Hv, device=DEV))
    offsets = _offsets(case, seed) if case["op"] != "step" else None
    seqs = case["seqs"] if offsets else B
    s["state"] = 0.3 * normal(seqs, Hv, dk, dv)
    if case["op"] == "step":
        for name in ("q", "k", "v", "g", "beta"):
            s[name] = s[name][:, 0].contiguous()
        s["state_out"] = torch.empty_like(s["state"])
        return s
    s["offsets"] = offsets
    s["cu"] = torch.tensor(offsets, dtype=torch.int32, device=DEV) if offsets else None
    if case["op"] == "train":
        s["do"], s["dstate"] = normal(B, T, Hv, dv).to(t), 0.1 * normal(seqs, Hv, dk, dv)
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------
def _orth(G, base, wide):
    t = G.dtype
    X = G.to(wide)
    tall = X.shape[-2] > X.shape[-1]
    X = X.mT if tall else X
    X = X / (X.square().sum((-2, -1), keepdim=True).sqrt() + EPS)
    a, b, c = COEF
    for _ in range(STEPS):
        A = X @ X.mT
        X = a * X + (b * A + c * (A @ A)) @ X
    X = X.mT if tall else X
    return (X if base is None else 0.99 * base.to(wide) - 0.02 * X).to(t)


def _to_rows(at, x):
    """(B, T, ...) or packed tokens -> (sequences, chunks * CHUNK, ...), zeros behind each sequence's end."""
    if at is None:
        pad = -x.shape[1] % CHUNK
        return torch.cat([x, x.new_zeros(x.shape[0], pad, *x.shape[2:])], 1) if pad else x
    at, live = at
    x = torch.cat([x[0], x.new_zeros(1, *x.shape[2:])])
    return x[torch.where(live, at, x.shape[0] - 1)]


def _from_rows(at, x, T):
    if at is None:
        return x[:, :T]
    at, live = at
    out = x.new_zeros(1, T, *x.shape[2:])
    out[0, at[live]] = x[live]
    return out


def _chunked(q, k, v, g, beta, S, scale):
    """The delta rule over (sequences, T, H, d) in float32, T a multiple of CHUNK: within a chunk one unit lower
    triangular system, from chunk to chunk the state."""
    R, T, H, dk = k.shape
    n = T // CHUNK

    def split(x):  # -> (R, H, n, CHUNK, d)
        return x.reshape(R, n, CHUNK, H, -1).permute(0, 3, 1, 2, 4)

    q, k, v, beta = split(q * scale), split(k), split(v), split(beta)
    # log decays summed in 64 bits: differences of long sums
    G = split(g.double()).cumsum(3)
    D = (G - G.mT).float()
    low = torch.ones(CHUNK, CHUNK, device=q.device).tril()
    D = torch.where(low.bool(), D, torch.zeros_like(D)).exp() * low
    N = ((k @ k.mT) * D).tril(-1)
    P = (q @ k.mT) * D
    A = N * beta.mT
    # rows of (I + A)^-1, one after the other
    rows = [torch.eye(CHUNK, device=q.device)[0].expand(*A.shape[:-2], CHUNK)]
    for i in range(1, CHUNK):
        done = torch.stack(rows, -2)
        row = torch.eye(CHUNK, device=q.device)[i] - (A[..., i : i + 1, :i] @ done)[..., 0, :]
        rows.append(row)
    inv = torch.stack(rows, -2)
    last = G[..., -1:, :]
    e, tail, keep = G.exp().float(), (last - G).exp().float(), last.exp().float()
    out = []
    for c in range(n):
        X = v[:, :, c] - e[:, :, c] * (k[:, :, c] @ S)
        U = beta[:, :, c] * (inv[:, :, c] @ X)
        out.append(e[:, :, c] * (q[:, :, c] @ S) + P[:, :, c] @ U)
        S = keep[:, :, c] * S + (tail[:, :, c] * k[:, :, c]).mT @ U
    o = torch.stack(out, 2).permute(0, 2, 3, 1, 4).reshape(R, T, H, -1) if out else v.new_zeros(R, 0, H, v.shape[-1])
    return o, S


def _delta(s, q, k, v, g, beta, S):
    case = s["case"]
    group = case["Hv"] // case["Hk"]
    at = None
    if s["offsets"] is not None:
        longest = max(b - a for a, b in zip(s["offsets"], s["offsets"][1:]))
        at = s["cu"][:-1, None] + torch.arange(-(-longest // CHUNK) * CHUNK, device=DEV)
        at = at, at < s["cu"][1:, None]
    q, k = (_to_rows(at, x).float().repeat_interleave(group, 2) for x in (q, k))
    o, S = _chunked(q, k, _to_rows(at, v).float(), _to_rows(at, g), _to_rows(at, beta), S, case["dk"] ** -0.5)
    return _from_rows(at, o, case["T"]).to(v.dtype), S


def _step(s):
    case = s["case"]
    group = case["Hv"] // case["Hk"]
    q, k = (x.float().repeat_interleave(group, 1) for x in (s["q"], s["k"]))
    S = s["state"] * s["g"].exp()[..., None, None]
    e = s["beta"][..., None] * (s["v"].float() - (k[..., None] * S).sum(-2))
    S = S + k[..., None] * e[..., None, :]
    return ((q[..., None] * S).sum(-2) * case["dk"] ** -0.5).to(s["v"].dtype), S


def run(state):
    s, case = state, state["case"]
    if own:
        return _run_own(s, case)
    if case["op"] == "orth":
        return _orth(s["G"], s["base"], torch.float64 if case["type"] == "f64" else torch.float32)
    if case["op"] == "step":
        return _step(s)
    args = [s[x] for x in ("q", "k", "v", "g", "beta", "state")]
    if case["op"] == "fwd":
        return _delta(s, *args)
    args = [x.detach().requires_grad_() for x in args]
    o, S = _delta(s, *args)
    return (o.detach(), S.detach(), *torch.autograd.grad([o, S], args, [s["do"], s["dstate"]]))


def _run_own(s, case):
    import gaussian_process_amd as gp

    if case["op"] == "orth":
        if s["base"] is None:
            return gp.orthogonalize(s["G"], steps=STEPS, coefficients=COEF, eps=EPS)
        return gp.orthogonalize(s["G"], steps=STEPS, coefficients=COEF, eps=EPS, alpha=-0.02, beta=0.99, base=s["base"])
    args = [s[x] for x in ("q", "k", "v", "g", "beta")]
    if case["op"] == "step":
        return gp.gated_delta_rule_step(*args, s["state"], state_out=s["state_out"])
    if case["op"] == "fwd":
        return gp.gated_delta_rule(*args, initial_state=s["state"], cu_seqlens=s["cu"])
    o, S, saved = gp.gated_delta_rule(*args, initial_state=s["state"], cu_seqlens=s["cu"], save_for_backward=True)
    return (o, S, *gp.gated_delta_rule_backward(saved, s["do"], s["dstate"]))


# ---- what a pass cannot do without ------------------------------------------------------------------------------
def work(case):
    z = SIZE[case["type"]]
    if case["op"] == "orth":
        small, large = sorted((case["n"], case["m"]))
        b = case["batch"]
        # X X^T and A A are symmetric: half of each is enough
        return {"flops": STEPS * b * small * small * (large + small + 2 * large),
                "bytes": b * small * large * z * (3 if case["base"] else 2)}
    Hk, Hv, dk, dv, B = case["Hk"], case["Hv"], case["dk"], case["dv"], case["B"]
    tokens = B * case.get("T", 1)
    states = (case.get("seqs") or B) * Hv * dk * dv * 4
    io = tokens * (2 * Hk * dk * z + 2 * Hv * dv * z + 2 * Hv * 4) + 2 * states
    if case["op"] != "train":
        # S^T k, the rank-one update and S^T q
        return {"flops": 6 * tokens * Hv * dk * dv, "bytes": io}
    # the gradients of q, k, v, g, beta and the first state; those of o and of the last state are read
    io += tokens * (2 * Hk * dk * z + 2 * Hv * dv * z + 2 * Hv * 4) + 2 * states
    return {"flops": 20 * tokens * Hv * dk * dv, "bytes": io}


# ---- from the definition, in 64 bits ----------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "orth":
        X = s["G"].double()
        flip = X.size(-2) > X.size(-1)
        if flip:
            X = X.transpose(-1, -2)
        X = X / (torch.linalg.matrix_norm(X, keepdim=True) + EPS)
        for _ in range(STEPS):
            gram = torch.matmul(X, X.transpose(-1, -2))
            once = torch.matmul(gram, X)
            X = COEF[0] * X + COEF[1] * once + COEF[2] * torch.matmul(gram, once)
        if flip:
            X = X.transpose(-1, -2)
        return X.contiguous() if s["base"] is None else 0.99 * s["base"].double() - 0.02 * X
    Hv, dk, dv = case["Hv"], case["dk"], case["dv"]
    group = Hv // case["Hk"]
    scale = 1.0 / math.sqrt(dk)
    if case["op"] == "step":
        q, k, v = (s[x].double() for x in "qkv")
        S = s["state"].double().clone()
        o = torch.empty(case["B"], Hv, dv, dtype=torch.float64, device=DEV)
        for h in range(Hv):
            M = S[:, h] * torch.exp(s["g"][:, h].double())[:, None, None]
            miss = v[:, h] - torch.bmm(k[:, None, h // group], M)[:, 0]
            M = M + s["beta"][:, h].double()[:, None, None] * k[:, h // group, :, None] * miss[:, None, :]
            S[:, h], o[:, h] = M, scale * torch.bmm(q[:, None, h // group], M)[:, 0]
        return o, S
    # token by token; all sequences and heads side by side, a sequence that has ended keeps its state
    off = s["offsets"] or [0, case["T"]]
    R, longest = s["state"].shape[0], max(b - a for a, b in zip(off, off[1:]))
    if case["op"] == "train" and longest * R * Hv * dk * dv * 8 > 60e9:
        return None

    def lay(x, heads):  # -> (longest, R, Hv, d)
        x = x.double().repeat_interleave(Hv // heads, 2)
        if s["offsets"] is None:
            return x.transpose(0, 1)
        y = x.new_zeros(longest, R, *x.shape[2:])
        for r in range(R):
            y[: off[r + 1] - off[r], r] = x[0, off[r] : off[r + 1]]
        return y

    def back(y):
        if s["offsets"] is None:
            return y.transpose(0, 1)
        return torch.cat([y[: off[r + 1] - off[r], r] for r in range(R)])[None]

    q, k, v = lay(s["q"], case["Hk"]), lay(s["k"], case["Hk"]), lay(s["v"], Hv)
    a, b = lay(s["g"], Hv).exp(), lay(s["beta"], Hv)
    S = s["state"].double()
    o, kept = torch.zeros_like(v), []
    for t in range(longest):
        kept.append(S if case["op"] == "train" else None)
        S = S * a[t][..., None, None]
        miss = v[t] - (k[t].unsqueeze(-2) @ S).squeeze(-2)
        S = torch.addcmul(S, k[t].unsqueeze(-1), (b[t].unsqueeze(-1) * miss).unsqueeze(-2))
        o[t] = scale * (q[t].unsqueeze(-2) @ S).squeeze(-2)
    if case["op"] == "fwd":
        return back(o), S
    do, dS = lay(s["do"], Hv), s["dstate"].double()
    dq, dk_, dv_, da, db = (torch.zeros_like(x) for x in (q, k, v, a, b))
    last = S
    for t in reversed(range(longest)):
        before = kept.pop()
        faded = before * a[t][..., None, None]
        miss = v[t] - (k[t].unsqueeze(-2) @ faded).squeeze(-2)
        dq[t] = scale * (last @ do[t].unsqueeze(-1)).squeeze(-1)
        dS = dS + scale * q[t].unsqueeze(-1) * do[t].unsqueeze(-2)
        down = (k[t].unsqueeze(-2) @ dS).squeeze(-2)
        db[t] = (down * miss).sum(-1)
        dmiss = b[t].unsqueeze(-1) * down
        dv_[t] = dmiss
        dk_[t] = b[t].unsqueeze(-1) * (dS @ miss.unsqueeze(-1)).squeeze(-1) - (faded @ dmiss.unsqueeze(-1)).squeeze(-1)
        dS = dS - k[t].unsqueeze(-1) * dmiss.unsqueeze(-2)
        da[t] = (dS * before).sum((-2, -1))
        dS = dS * a[t][..., None, None]
        last = before

    def shared(x):
        x = back(x)
        return x.reshape(*x.shape[:2], case["Hk"], group, -1).sum(3)

    return back(o), S, shared(dq), shared(dk_), back(dv_), back(da * a), back(db), dS


if __name__ == "__main__":
    for c in listed():
        w = work(c)
        print("%-28s %10.3g bytes %10.3g flops" % (c["name"], w["bytes"], w["flops"]))

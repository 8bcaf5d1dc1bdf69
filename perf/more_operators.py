"""The gated delta rule and the verification of drafted tokens, as cases to be
timed: a linear-attention layer's training step, its reading of a prompt, its
decode step (one token, or a block of drafted ones, over a pool of states), and
what a serving loop does with the drafts' logits.

``run`` is the plain form (elementary torch operations in float32, the chunked
form of the recurrence) or, where ``own`` is true, the calls of ``rwkv7m_amd``.
``exact`` is the definition in float64, token by token.  Widths and heads are
those of the 0.185B, 1B and 7B models (768, 2048, 4096 in heads of 64 or 128)
or generic; 65536 is the size of the RWKV world tokenizer's embedding, 65529
its tokens.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}
CHUNK = 64  # of the plain form


def listed():
    return [
        # one new token of a 0.185B-sized model: nothing but latency
        dict(name="step_token", op="step", dtype="bf16", gtype="f32", B=1,
             T=1, Hk=12, Hv=12, Dk=64, Dv=64, slots=1, ragged=False,
             update=True),
        # a serving batch's decode step over a pool of states, value heads in
        # pairs on a key head: the state's bytes are all there is
        dict(name="step_batch", op="step", dtype="bf16", gtype="f32", B=192,
             T=1, Hk=16, Hv=32, Dk=128, Dv=128, slots=256, ragged=False,
             update=True),
        # a block of drafted tokens read before it is verified: outputs
        # alone, the states stay
        dict(name="step_drafts", op="step", dtype="bf16", gtype="bf16", B=48,
             T=6, Hk=32, Hv=32, Dk=64, Dv=64, slots=64, ragged=True,
             update=False),
        # a prompt of odd length, one sequence: few heads, many tokens
        dict(name="prompt_one", op="rule", train=False, dtype="bf16",
             gtype="f32", B=1, T=1999, Hk=16, Hv=32, Dk=128, Dv=128,
             state=False, fused=True),
        # short prompts continued from states, float32, odd sizes
        dict(name="prompt_f32", op="rule", train=False, dtype="f32",
             gtype="f32", B=3, T=333, Hk=12, Hv=12, Dk=64, Dv=72, state=True,
             fused=False),
        # a training step at the 0.185B model's width
        dict(name="train_0185b", op="rule", train=True, dtype="bf16",
             gtype="f32", B=8, T=512, Hk=12, Hv=12, Dk=64, Dv=64,
             state=False, fused=True),
        # the same at a 1B model's width and full context: the largest
        dict(name="train_1b", op="rule", train=True, dtype="bf16",
             gtype="f32", B=8, T=4096, Hk=16, Hv=16, Dk=128, Dv=128,
             state=False, fused=False),
        # a segment of a longer sequence: state and its gradient carried,
        # value heads in threes on a key head, odd length
        dict(name="train_carry", op="rule", train=True, dtype="bf16",
             gtype="bf16", B=2, T=1001, Hk=8, Hv=24, Dk=96, Dv=128,
             state=True, fused=True),
        # float32 training
        dict(name="train_f32", op="rule", train=True, dtype="f32",
             gtype="f32", B=2, T=512, Hk=12, Hv=12, Dk=64, Dv=64, state=True,
             fused=False),
        # four drafts of one sequence
        dict(name="verify_one", op="verify", dtype="bf16", B=1, K=4, V=65536,
             temp=1.0, ragged=False, certain=False),
        # a serving batch's, ragged
        dict(name="verify_batch", op="verify", dtype="bf16", B=96, K=5,
             V=65536, temp=0.8, ragged=True, certain=False),
        # drafts found by lookup (no draft model), float32 logits
        dict(name="verify_lookup", op="verify", dtype="f32", B=24, K=8,
             V=65529, temp=1.0, ragged=True, certain=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo),
                                                      math.log(hi))))))


def draw(rng):
    op = rng.choice(("step", "rule", "rule", "verify"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    if op == "verify":
        V = rng.choice((65536, 65529, _log(rng, 300, 131072),
                        _log(rng, 300, 131072)))
        K = rng.randint(1, 12)
        most = (96 * 11 * 65536 * 2) // ((2 * K + 1) * V * BYTES[dtype])
        return dict(op=op, dtype=dtype, B=_log(rng, 1, max(1, min(256, most))),
                    K=K, V=V, temp=rng.choice((1.0, 1.0, 0.7, 1.3)),
                    ragged=rng.random() < 0.5, certain=rng.random() < 0.3)
    Dk, Dv = rng.choice(((64, 64), (128, 128), (64, 128), (128, 256),
                         (8 * rng.randint(2, 16), 8 * rng.randint(2, 32))))
    groups = rng.choice((1, 1, 2, 3, 4))
    gtype = rng.choice(("f32", dtype))
    c = dict(op=op, dtype=dtype, gtype=gtype, Dk=Dk, Dv=Dv)
    if op == "step":
        Hk = _log(rng, 1, 64 // groups)
        most = (192 * 32 * 128 * 128) // (Hk * groups * Dk * Dv)
        B = _log(rng, 1, max(1, min(256, most)))
        T = rng.choice((1, 1, rng.randint(2, 8)))
        return dict(c, B=B, T=T, Hk=Hk, Hv=Hk * groups,
                    slots=B + rng.randint(0, B), ragged=rng.random() < 0.5,
                    update=rng.random() < 0.7)
    train = rng.random() < 0.5
    Hk = _log(rng, 1, 32 // groups)
    per = Hk * groups * (Dk + Dv) * (4 if dtype == "f32" else 1)
    most = (8 * 4096 * 16 * 256) // per
    T = _log(rng, 1, min(8192, most))
    B = _log(rng, 1, max(1, min(16, most // T)))
    return dict(c, train=train, B=B, T=T, Hk=Hk, Hv=Hk * groups,
                state=rng.random() < 0.5, fused=rng.random() < 0.5)


# --- inputs ---------------------------------------------------------------

def _vectors(c, g):
    """q, k (of length 1 in each head), v, the log decays and betas, as a
    layer's projections give them: ``fused`` ones are views of one."""
    B, T, Hk, Hv, Dk, Dv = (c[n] for n in ("B", "T", "Hk", "Hv", "Dk", "Dv"))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    q, k, v = normal(B, T, Hk, Dk), normal(B, T, Hk, Dk), normal(B, T, Hv, Dv)
    # keys of a head resemble each other, the more the nearer
    k = k + 0.7 * normal(B, 1, Hk, Dk)
    q, k = (x / x.square().sum(-1, keepdim=True).sqrt() for x in (q, k))
    # heads that forget within a few tokens and heads that hardly do
    rate = torch.exp(math.log(0.002) + math.log(1000.0) * torch.rand(
        Hv, generator=g, device=DEV))
    decay = -rate * torch.nn.functional.softplus(normal(B, T, Hv))
    beta = torch.sigmoid(normal(B, T, Hv))
    dt, gt = DT[c["dtype"]], DT[c["gtype"]]
    q, k, v = q.to(dt), k.to(dt), v.to(dt)
    if c.get("fused"):
        one = torch.cat([x.reshape(B, T, -1) for x in (q, k, v)], -1)
        q = one[..., :Hk * Dk].view(B, T, Hk, Dk)
        k = one[..., Hk * Dk:2 * Hk * Dk].view(B, T, Hk, Dk)
        v = one[..., 2 * Hk * Dk:].view(B, T, Hv, Dv)
    return dict(q=q, k=k, v=v, g=decay.to(gt), beta=beta.to(gt))


def prepare(case, seed):
    """The tensors a program holds before the call."""
    c = case
    g = torch.Generator(DEV).manual_seed(seed)
    if c["op"] == "verify":
        return _prepare_verify(c, g)
    s = dict(_vectors(c, g), case=c)
    B, T, Hv, Dk, Dv = (c[n] for n in ("B", "T", "Hv", "Dk", "Dv"))

    def states(n):
        return 0.3 * torch.randn(n, Hv, Dv, Dk, generator=g, device=DEV)

    if c["op"] == "step":
        s["state"] = states(c["slots"])
        s["slots"] = torch.randperm(c["slots"], generator=g, device=DEV)[:B]
        s["lengths"] = (torch.randint(0, T + 1, (B,), generator=g, device=DEV)
                        if c["ragged"] else None)
        return s
    s["initial"] = states(B) if c["state"] else None
    if c["train"]:
        s["do"] = torch.randn(B, T, Hv, Dv, generator=g, device=DEV).to(
            DT[c["dtype"]])
        s["dstate"] = states(B) if c["state"] else None
        for n in ("q", "k", "v", "g", "beta", "initial"):
            if s[n] is not None:
                s[n] = s[n].detach().requires_grad_()
    return s


def _prepare_verify(c, g):
    B, K, V = c["B"], c["K"], c["V"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    x = 2.0 * normal(B, K + 1, V)
    at = torch.randint(0, V, (B, K + 1, 4), generator=g, device=DEV)
    x.scatter_(-1, at, 9.0 + 2.0 * normal(B, K + 1, 4))
    # the draft model's opinion, and a token drawn from it by the race of
    # exponentials
    y = x[:, :K] + 0.5 * normal(B, K, V)
    race = torch.rand(B, K, V, generator=g, device=DEV).clamp_(min=1e-20)
    tokens = (y / c["temp"] - race.log_().neg_().log_()).argmax(-1)
    s = dict(case=c, tokens=tokens,
             accept=torch.rand(B, K, generator=g, device=DEV),
             sample=torch.rand(B, generator=g, device=DEV),
             drafted=(torch.randint(0, K + 1, (B,), generator=g, device=DEV)
                      if c["ragged"] else None))
    s["target"] = x.to(DT[c["dtype"]])
    s["draft"] = None if c["certain"] else y.to(DT[c["dtype"]])
    return s


# --- the plain forms ------------------------------------------------------

def _chunks(x, n, C):
    """[B, T, H, ...] as float32 [B, H, n, C, ...], zeros behind T."""
    x = x.detach().float().transpose(1, 2)
    pad = n * C - x.shape[2]
    if pad:
        x = torch.cat([x, x.new_zeros(*x.shape[:2], pad, *x.shape[3:])], 2)
    return x.reshape(*x.shape[:2], n, C, *x.shape[3:]).contiguous()


def _tokens(x, T):
    """Back to [B, T, H, ...]."""
    x = x.reshape(x.shape[0], x.shape[1], -1, *x.shape[4:])[:, :, :T]
    return x.transpose(1, 2)


def _tr(x):
    return x.transpose(-1, -2).contiguous()


def _plain_rule(s):
    c = s["case"]
    B, T, Hk, Hv, Dk, Dv = (c[n] for n in ("B", "T", "Hk", "Hv", "Dk", "Dv"))
    per, scale, C = Hv // Hk, Dk ** -0.5, CHUNK
    n = -(-T // C)
    dev = s["q"].device
    q, k = (_chunks(s[x], n, C).repeat_interleave(per, 1) for x in "qk")
    v, b = _chunks(s["v"], n, C), _chunks(s["beta"], n, C)[..., None]
    # far tokens' decays: differences of sums in 64 bits
    G = _chunks(s["g"], n, C).double().cumsum(-1)
    i = torch.arange(C, device=dev)
    low = i[:, None] >= i
    E = torch.where(low, G[..., :, None] - G[..., None, :], 0.0).exp().float()
    E = E * low
    strict = (i[:, None] > i).float()
    first = G.exp().float()[..., None]               # e^G
    last = (G[..., -1:] - G).exp().float()[..., None]  # e^(G_L - G)
    whole = G[..., -1].exp().float()[..., None, None]  # e^G_L
    A = (k @ _tr(k)) * E * strict * b
    P = (q @ _tr(k)) * E
    # the inverse of I + A, row by row
    inv = torch.eye(C, device=dev).expand_as(A).contiguous()
    for t in range(1, C):
        inv[..., t, :t] = -(A[..., t, :t, None] * inv[..., :t, :t]).sum(-2)
    S = (torch.zeros(B, Hv, Dv, Dk, device=dev) if s["initial"] is None
         else s["initial"].detach())
    S0, X = [], []
    for j in range(n):
        S0.append(S)
        R = b[:, :, j] * (v[:, :, j] - first[:, :, j] * (k[:, :, j] @ _tr(S)))
        X.append(inv[:, :, j] @ R)
        S = whole[:, :, j] * S + _tr(last[:, :, j] * X[-1]) @ k[:, :, j]
    S0, X = torch.stack(S0, 2), torch.stack(X, 2)
    o = scale * (first * (q @ _tr(S0)) + P @ X)
    dt, gt = s["q"].dtype, s["g"].dtype
    out = [_tokens(o, T).to(dt), S]
    if not c["train"]:
        return out
    do = _chunks(s["do"], n, C)
    D = torch.zeros_like(S) if s["dstate"] is None else s["dstate"]
    dX = scale * (_tr(P) @ do)
    carry = scale * (_tr(first * do) @ q)
    invT = _tr(inv)
    Ds, dR = [None] * n, [None] * n
    for j in reversed(range(n)):
        Ds[j] = D
        y = dX[:, :, j] + last[:, :, j] * (k[:, :, j] @ _tr(D))
        dR[j] = invT[:, :, j] @ y
        D = (whole[:, :, j] * D + carry[:, :, j]
             - _tr(b[:, :, j] * first[:, :, j] * dR[j]) @ k[:, :, j])
    D_end, dR = torch.stack(Ds, 2), torch.stack(dR, 2)
    dA = -(dR @ _tr(X)) * strict * E
    dP = scale * (do @ _tr(X)) * E
    dq = scale * first * (do @ S0) + dP @ k
    left = dA @ k - first * (dR @ S0)
    right = _tr(dP) @ q + _tr(b * dA) @ k + (last * X) @ D_end
    db = (k * left).sum(-1) + (dR * v).sum(-1)
    dG = ((q * dq).sum(-1) + b[..., 0] * (k * left).sum(-1)
          - (k * right).sum(-1)).double()
    S_end = whole * S0 + _tr(last * X) @ k
    dG[..., -1] += (D_end * S_end).sum((-1, -2))
    dg = dG.flip(-1).cumsum(-1).flip(-1)

    def grouped(x):
        return x.reshape(B, Hk, per, *x.shape[2:]).sum(2)

    out += [_tokens(grouped(dq), T).to(dt),
            _tokens(grouped(b * left + right), T).to(dt),
            _tokens(b * dR, T).to(dt), _tokens(dg, T).to(gt),
            _tokens(db, T).to(gt)]
    return out + ([D] if s["initial"] is not None else [])


def _plain_step(s):
    c = s["case"]
    per, scale = c["Hv"] // c["Hk"], c["Dk"] ** -0.5
    q, k = (s[x].float().repeat_interleave(per, 2) for x in "qk")
    v, a, b = s["v"].float(), s["g"].float().exp(), s["beta"].float()
    S = s["state"][s["slots"]]
    o = torch.zeros_like(v)
    for t in range(c["T"]):
        S1 = S * a[:, t, :, None, None]
        off = v[:, t] - (S1 * k[:, t, :, None, :]).sum(-1)
        S1 = S1 + (b[:, t, :, None] * off)[..., None] * k[:, t, :, None, :]
        o1 = scale * (S1 * q[:, t, :, None, :]).sum(-1)
        if s["lengths"] is None:
            S, o[:, t] = S1, o1
        else:
            on = (s["lengths"] > t)[:, None, None]
            S, o[:, t] = torch.where(on[..., None], S1, S), on * o1
    if not c["update"]:
        return [o.to(s["v"].dtype)]
    return [o.to(s["v"].dtype), s["state"].index_copy_(0, s["slots"], S)]


def _plain_verify(s):
    c = s["case"]
    B, K, V = c["B"], c["K"], c["V"]
    at = s["tokens"][..., None]
    # 64 bits: a sampled token lies next to the border of a sum over V
    p = s["target"].double() / c["temp"]
    p = (p - p.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    if s["draft"] is None:
        q = torch.zeros_like(p[:, :K]).scatter_(-1, at, 1.0)
    else:
        q = s["draft"].double() / c["temp"]
        q = (q - q.amax(-1, keepdim=True)).exp()
        q = q / q.sum(-1, keepdim=True)
    px, qx = p[:, :K].gather(-1, at)[..., 0], q.gather(-1, at)[..., 0]
    i = torch.arange(K + 1, device=p.device)
    n = s["drafted"] if s["drafted"] is not None else i.new_full((B,), K)
    given = i[:K] < n[:, None]
    took = given & (s["accept"].double() * qx < px)
    m = took.long().cumprod(-1).sum(-1)
    rest = p[torch.arange(B, device=p.device), m]
    last = torch.cat([q, q.new_zeros(B, 1, V)], 1)[
        torch.arange(B, device=p.device), m]
    rest = torch.where((m < n)[:, None], (rest - last).clamp(min=0.0), rest)
    cum = rest.cumsum(-1)
    new = (cum <= s["sample"].double()[:, None] * cum[:, -1:]).sum(-1)
    drafts = torch.cat([s["tokens"], new[:, None]], 1)
    out = torch.where(i < m[:, None], drafts, -1)
    out.scatter_(1, m[:, None], new[:, None])
    prob = torch.where(given, (px / qx).clamp(max=1.0), 0.0)
    return [out, m, prob.float()]


def _own_run(s):
    import rwkv7m_amd
    c = s["case"]
    if c["op"] == "verify":
        return list(rwkv7m_amd.verify_drafts(
            s["target"], s["tokens"], s["draft"], s["accept"], s["sample"],
            draft_lengths=s["drafted"], temperature=c["temp"]))
    vectors = [s[n] for n in ("q", "k", "v", "g", "beta")]
    if c["op"] == "step":
        o = rwkv7m_amd.gated_delta_step(
            *vectors, s["state"], lengths=s["lengths"], slots=s["slots"],
            update_state=c["update"])
        return [o, s["state"]] if c["update"] else [o]
    if not c["train"]:
        with torch.no_grad():
            return list(rwkv7m_amd.gated_delta_rule(*vectors, s["initial"]))
    o, end = rwkv7m_amd.gated_delta_rule(*vectors, s["initial"])
    if s["initial"] is None:
        return [o, end, *torch.autograd.grad(o, vectors, s["do"])]
    return [o, end, *torch.autograd.grad(
        (o, end), [*vectors, s["initial"]], (s["do"], s["dstate"]))]


def run(state):
    """One pass, as a program calls it."""
    if own:
        return _own_run(state)
    with torch.no_grad():
        return {"rule": _plain_rule, "step": _plain_step,
                "verify": _plain_verify}[state["case"]["op"]](state)


# --- what a pass cannot do without ----------------------------------------

def work(case):
    """Bytes: each input read once and each output written once.  Operations:
    those of the recurrence, three products of a vector with the state a
    token and head, and seven more for the gradients."""
    c, eb = case, BYTES[case["dtype"]]
    if c["op"] == "verify":
        rows = c["B"] * (c["K"] + 1 + (0 if c["certain"] else c["K"]))
        return {"bytes": rows * c["V"] * eb + c["B"] * (c["K"] + 1) * 24,
                "flops": 4 * rows * c["V"]}
    B, T, Hk, Hv, Dk, Dv = (c[n] for n in ("B", "T", "Hk", "Hv", "Dk", "Dv"))
    qk, v = 2 * B * T * Hk * Dk * eb, B * T * Hv * Dv * eb
    gates, state = 2 * B * T * Hv * BYTES[c["gtype"]], B * Hv * Dk * Dv * 4
    flops = 6 * B * T * Hv * Dk * Dv
    if c["op"] == "step":
        return {"bytes": qk + 2 * v + gates + state * (1 + c["update"]),
                "flops": flops}
    first = state * (1 if c["state"] else 0)
    if not c["train"]:
        return {"bytes": qk + 2 * v + gates + state + first, "flops": flops}
    # q, k, v, do; o, dq, dk, dv; gates and their gradients; states, theirs
    return {"bytes": 2 * qk + 4 * v + 2 * gates + state + 3 * first,
            "flops": flops * 20 // 6}


# --- the definition in float64 --------------------------------------------

def _exact_vectors(s):
    """[T, B, Hv, ...] in float64, key heads repeated."""
    per = s["case"]["Hv"] // s["case"]["Hk"]
    q, k = (s[n].detach().double().repeat_interleave(per, 2) for n in "qk")
    v, g, b = (s[n].detach().double() for n in ("v", "g", "beta"))
    return [x.transpose(0, 1).contiguous() for x in (q, k, v, g.exp(), b)]


def _advance(S, k, v, a, b):
    """S (I - b k k^T) a + b v k^T of one token."""
    Sk = torch.einsum("bhij,bhj->bhi", S, k)
    u = b[..., None] * (v - a[..., None] * Sk)
    return a[..., None, None] * S + u[..., :, None] * k[..., None, :], Sk, u


def _exact_rule(s):
    c = s["case"]
    B, T, Hk, Hv, Dk, Dv = (c[n] for n in ("B", "T", "Hk", "Hv", "Dk", "Dv"))
    scale, per = Dk ** -0.5, Hv // Hk
    q, k, v, a, b = _exact_vectors(s)
    S = (torch.zeros(B, Hv, Dv, Dk, dtype=torch.float64, device=q.device)
         if s["initial"] is None else s["initial"].detach().double())
    part = max(1, math.isqrt(T))
    o, kept = torch.empty_like(v), []
    for t in range(T):
        if c["train"] and t % part == 0:
            kept.append(S)
        S, _, _ = _advance(S, k[t], v[t], a[t], b[t])
        o[t] = scale * torch.einsum("bhij,bhj->bhi", S, q[t])
    out = [o.transpose(0, 1), S]
    if not c["train"]:
        return out
    do = s["do"].double().transpose(0, 1)
    D = (torch.zeros_like(S) if s["dstate"] is None
         else s["dstate"].double().clone())
    dq, dk, dv, dg, db = (torch.empty_like(x) for x in (q, k, v, a, b))
    for j in reversed(range(len(kept))):
        S, steps = kept[j], []
        for t in range(j * part, min(T, (j + 1) * part)):
            S1, Sk, u = _advance(S, k[t], v[t], a[t], b[t])
            steps.append((t, S, Sk, u, S1))
            S = S1
        for t, S, Sk, u, S1 in reversed(steps):
            dq[t] = scale * torch.einsum("bhij,bhi->bhj", S1, do[t])
            D = D + scale * do[t][..., :, None] * q[t][..., None, :]
            du = torch.einsum("bhij,bhj->bhi", D, k[t])
            db[t] = (du * (v[t] - a[t][..., None] * Sk)).sum(-1)
            dv[t] = b[t][..., None] * du
            dSk = -(a[t] * b[t])[..., None] * du
            dg[t] = a[t] * ((D * S).sum((-1, -2))
                            - b[t] * (du * Sk).sum(-1))
            dk[t] = (torch.einsum("bhij,bhi->bhj", D, u)
                     + torch.einsum("bhij,bhi->bhj", S, dSk))
            D = (a[t][..., None, None] * D
                 + dSk[..., :, None] * k[t][..., None, :])

    def back(x):
        return x.transpose(0, 1)

    def grouped(x):
        return back(x).reshape(B, T, Hk, per, Dk).sum(3)

    out += [grouped(dq), grouped(dk), back(dv), back(dg), back(db)]
    return out + ([D] if s["initial"] is not None else [])


def _exact_step(s):
    c = s["case"]
    q, k, v, a, b = _exact_vectors(s)
    pool, o = s["state"].double(), torch.zeros_like(v)
    S = pool[s["slots"]]
    n = s["lengths"]
    if n is None:
        n = torch.full((c["B"],), c["T"], device=q.device)
    for t in range(c["T"]):
        live = n > t
        S = S.clone()
        S[live] = _advance(S[live], k[t][live], v[t][live], a[t][live],
                           b[t][live])[0]
        o[t][live] = torch.einsum("bhij,bhj->bhi", S[live],
                                  q[t][live]) * c["Dk"] ** -0.5
    out = [o.transpose(0, 1)]
    if c["update"]:
        pool[s["slots"]] = S
        out.append(pool)
    return out


def _exact_verify(s):
    c = s["case"]
    prob = torch.zeros(c["B"], c["K"], dtype=torch.float64,
                       device=s["target"].device)
    for i in range(c["K"]):
        x = s["tokens"][:, i:i + 1]
        lp = torch.log_softmax(s["target"][:, i].double() / c["temp"], -1)
        lp = lp.gather(-1, x)[:, 0]
        if s["draft"] is not None:
            lq = torch.log_softmax(s["draft"][:, i].double() / c["temp"], -1)
            lp = lp - lq.gather(-1, x)[:, 0]
        prob[:, i] = lp.clamp(max=0.0).exp()
        if s["drafted"] is not None:
            prob[:, i] *= s["drafted"] > i
    return [None, None, prob]


def exact(case, seed):
    s = prepare(case, seed)
    return {"rule": _exact_rule, "step": _exact_step,
            "verify": _exact_verify}[case["op"]](s)

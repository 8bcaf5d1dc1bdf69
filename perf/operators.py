"""The operators around a language model's head, as cases to be timed: the
layer norm before it (and before each block's mixes), the log probabilities,
entropy and top alternatives read from its logits, and the distillation loss
from a teacher's top logits.

``run`` is the plain form (elementary torch operations in float32) or, where
``own`` is true, the calls of ``rwkv7m_amd``.  ``exact`` is the definition in
float64.  65536 is the size of the RWKV world tokenizer's embedding, 65529 its
tokens; widths are those of the 0.185B, 1B and 7B models, or generic.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}


def listed():
    return [
        # the norm of one new token's hidden state: nothing but latency
        dict(name="norm_token", op="norm", train=False, dtype="bf16",
             ptype="bf16", rows=1, C=768),
        # a prompt of odd length read by a 7B model with fp32 parameters
        dict(name="norm_prompt", op="norm", train=False, dtype="bf16",
             ptype="f32", rows=1999, C=4096),
        # a norm in the training step of a 0.185B model
        dict(name="norm_train_0185b", op="norm", train=True, dtype="bf16",
             ptype="f32", rows=8 * 512, C=768),
        # the same of a 1B model at its full context: the largest norm
        dict(name="norm_train_1b", op="norm", train=True, dtype="bf16",
             ptype="f32", rows=8 * 4096, C=2048),
        # float32 training at a width that is no multiple of a vector
        dict(name="norm_train_odd", op="norm", train=True, dtype="f32",
             ptype="f32", rows=2731, C=1001),
        # one decoded token with its alternatives, under a grammar's mask
        dict(name="score_token", op="score", train=False, dtype="bf16", B=1,
             T=1, V=65536, K=20, temp=1.0, ignored=0.0, masked=0.5,
             shifted=False),
        # a serving batch's decode step in float32
        dict(name="score_batch", op="score", train=False, dtype="f32", B=96,
             T=1, V=65529, K=5, temp=0.7, ignored=0.0, masked=0.0,
             shifted=False),
        # prompts scored for an evaluation: the logits of each position
        # against the next token, a third of them context that is not scored
        dict(name="score_prompts", op="score", train=False, dtype="bf16",
             B=8, T=512, V=65536, K=10, temp=1.0, ignored=0.3, masked=0.0,
             shifted=True),
        # the policy's log probabilities and entropy bonus in a training
        # step: the gradient of both, odd vocabulary
        dict(name="score_train", op="score", train=True, dtype="bf16", B=4,
             T=511, V=65529, K=0, temp=1.0, ignored=0.2, masked=0.0,
             shifted=False),
        # one short sequence distilled: a launch of half the chip
        dict(name="distill_small", op="distill", dtype="bf16", B=1, T=128,
             V=65536, K=16, temp=1.0, ignored=0.0, shifted=False),
        # a 0.185B student's step: padding left out, the last position has
        # no target
        dict(name="distill_0185b", op="distill", dtype="bf16", B=8, T=512,
             V=65536, K=64, temp=2.0, ignored=0.1, shifted=True),
        # float32 logits over an odd vocabulary
        dict(name="distill_f32", op="distill", dtype="f32", B=3, T=333,
             V=32003, K=50, temp=1.5, ignored=0.1, shifted=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo),
                                                      math.log(hi))))))


def draw(rng):
    op = rng.choice(("norm", "score", "distill"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    if op == "norm":
        C = rng.choice((768, 1024, 2048, 4096, _log(rng, 16, 8192),
                        _log(rng, 16, 8192)))
        most = min(1 << 16, (8 * 4096 * 2048 * 2) // (C * BYTES[dtype]))
        return dict(op=op, train=rng.random() < 0.6, dtype=dtype,
                    ptype=rng.choice(("f32", "bf16")),
                    rows=_log(rng, 1, most), C=C)
    V = rng.choice((65536, 65529, _log(rng, 300, 131072),
                    _log(rng, 300, 131072)))
    most = (8 * 512 * 65536 * 2) // (V * BYTES[dtype])
    shifted = rng.random() < 0.4
    T = _log(rng, 2 if shifted else 1, max(2, min(2048, most)))
    B = _log(rng, 1, max(1, min(64, most // T)))
    c = dict(op=op, dtype=dtype, B=B, T=T, V=V,
             temp=rng.choice((1.0, 1.0, 0.7, 2.0)),
             ignored=rng.choice((0.0, 0.1, 0.5)), shifted=shifted)
    if op == "distill":
        return dict(c, K=_log(rng, 1, 128))
    train = rng.random() < 0.4
    return dict(c, train=train, K=0 if train else
                rng.choice((0, 1, 5, 20, rng.randint(1, 64))),
                masked=0.0 if train else rng.choice((0.0, 0.5, 0.999)))


# --- inputs ---------------------------------------------------------------

def _rows(c):
    return c["B"] * (c["T"] - 1 if c["shifted"] else c["T"])


def _left_out(c):
    return int(_rows(c) * c["ignored"])


def _logits(c, g):
    """[B, T, V] logits with the spread of a trained head's, and the view of
    them that has a target (all positions, or all but each row's last)."""
    x = torch.randn(c["B"], c["T"], c["V"], generator=g, device=DEV)
    x = x.mul_(2.0).to(DT[c["dtype"]])
    # a few likely tokens in each position
    at = torch.randint(0, c["V"], (c["B"], c["T"], 4), generator=g,
                       device=DEV)
    up = 6.0 + 3.0 * torch.randn(c["B"], c["T"], 4, generator=g, device=DEV)
    x.scatter_(-1, at, up.to(x.dtype))
    if c.get("masked", 0.0):
        keep = torch.rand(c["V"], generator=g, device=DEV) >= c["masked"]
        keep[g.initial_seed() % c["V"]] = True
        x.masked_fill_(~keep, float("-inf"))
    view = x[:, :-1] if c["shifted"] else x
    return view, at[:, :view.shape[1]]


def prepare(case, seed):
    """The tensors a program holds before the call."""
    c = case
    g = torch.Generator(DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    if c["op"] == "norm":
        dt, pt, C = DT[c["dtype"]], DT[c["ptype"]], c["C"]
        # the residual stream: some channels are far larger than the rest,
        # and a row has a mean
        x = normal(c["rows"], C) * (1.0 + normal(C).abs()) + 0.5 * normal(C)
        s = dict(case=c, x=x.to(dt), w=(1.0 + 0.1 * normal(C)).to(pt),
                 b=(0.1 * normal(C)).to(pt))
        if c["train"]:
            s["dy"] = (normal(c["rows"], C) + 0.3 * normal(C)).to(dt)
            for n in ("x", "w", "b"):
                s[n].requires_grad_()
        return s
    x, likely = _logits(c, g)
    s = dict(case=c, x=x)
    shape = x.shape[:2]
    out = torch.zeros(_rows(c), dtype=torch.bool, device=DEV)
    out[torch.randperm(_rows(c), generator=g, device=DEV)[:_left_out(c)]] = \
        True
    out = out.view(shape)
    if c["op"] == "score":
        tok = torch.randint(0, c["V"], shape, generator=g, device=DEV)
        pick = torch.rand(shape, generator=g, device=DEV) < 0.7
        s["tokens"] = torch.where(pick, likely[..., 0], tok).masked_fill(
            out, -100)
        if c["train"]:
            # an advantage for each scored token, and the bonus's weight
            s["g_lp"] = normal(*shape).masked_fill(out, 0.0) / _rows(c)
            s["g_ent"] = torch.full(shape, -0.01 / _rows(c),
                                    device=DEV).masked_fill(out, 0.0)
            s["x"] = x.requires_grad_()
        return s
    K = c["K"]
    # the teacher's top: its logits are the student's with another opinion,
    # some positions with fewer alternatives than the others
    ids = torch.empty(*shape, K, dtype=torch.int64, device=DEV)
    top = torch.empty(*shape, K, device=DEV)
    for i in range(shape[0]):
        top[i], ids[i] = (x[i].float() + normal(*x.shape[1:])).topk(K, -1)
    few = torch.rand(shape, generator=g, device=DEV) < 0.2
    short = torch.arange(K, device=DEV) >= (K + 1) // 2
    ids.masked_fill_(few[..., None] & short, -1)
    s["ids"], s["top"] = ids, top.to(DT[c["dtype"]])
    s["w"] = (~out).float() / max(1, _rows(c) - _left_out(c))
    s["x"] = x.requires_grad_()
    return s


# --- the plain forms ------------------------------------------------------

def _plain_norm(s):
    c, dt = s["case"], s["x"].dtype
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    dev = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((dev * dev).mean(-1, keepdim=True) + 1e-5)
    xh = dev * rstd
    y = (xh * w + b).to(dt)
    if not c["train"]:
        return [y]
    dy = s["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True)
                 - xh * (g * xh).mean(-1, keepdim=True))
    return [y, dx.to(dt), (dy * xh).sum(0).to(s["w"].dtype),
            dy.sum(0).to(s["b"].dtype)]


def _plain_top(x, k):
    """Ids of the k largest, equal ones in the order of their ids: a key of
    the value's bits in order above the id's complement."""
    bits = (x + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long()
    last = x.shape[-1] - 1
    key = order * (1 << 32) + (last - torch.arange(last + 1, device=DEV))
    return last - (key.topk(k, -1).values & 0xffffffff)


def _plain_score(s):
    c, tok = s["case"], s["tokens"]
    x = s["x"].float()
    z = x / c["temp"]
    z = z - z.amax(-1, keepdim=True)
    logp = z - z.exp().sum(-1, keepdim=True).log()
    p = logp.exp()
    plogp = torch.where(p > 0, p * logp, 0.0)
    ent = -plogp.sum(-1)
    at, scored = tok.clamp(min=0)[..., None], tok >= 0
    lp = torch.where(scored, logp.gather(-1, at)[..., 0], 0.0)
    if c["train"]:
        glp = (s["g_lp"] * scored)[..., None]
        d = -p * glp - s["g_ent"][..., None] * (plogp + p * ent[..., None])
        d.scatter_add_(-1, at, glp)
        return [lp, ent, (d / c["temp"]).to(s["x"].dtype)]
    if not c["K"]:
        return [lp, ent]
    ids = _plain_top(x, c["K"])
    return [lp, ent, ids, logp.gather(-1, ids)]


def _plain_distill(s):
    c, ids, w = s["case"], s["ids"], s["w"]
    T = c["temp"]
    t = (s["top"].float() / T).masked_fill(ids < 0, float("-inf"))
    t = t - t.amax(-1, keepdim=True)
    logq = t - t.exp().sum(-1, keepdim=True).log()
    q = logq.exp()
    z = s["x"].float() / T
    z = z - z.amax(-1, keepdim=True)
    logp = z - z.exp().sum(-1, keepdim=True).log()
    at = ids.clamp(min=0)
    kl = torch.where(q > 0, q * (logq - logp.gather(-1, at)), 0.0).sum(-1)
    rows = torch.where(w != 0, T * T * kl, 0.0)
    wt = (w * T)[..., None]
    d = logp.exp() * wt
    d.scatter_add_(-1, at, -q * wt)
    return [(w * rows).sum(), rows, d.to(s["x"].dtype)]


def _own_run(s):
    import rwkv7m_amd
    c = s["case"]
    if c["op"] == "norm":
        if not c["train"]:
            with torch.no_grad():
                return [rwkv7m_amd.layer_norm(s["x"], s["w"], s["b"])]
        y = rwkv7m_amd.layer_norm(s["x"], s["w"], s["b"])
        return [y, *torch.autograd.grad(y, [s["x"], s["w"], s["b"]],
                                        s["dy"])]
    if c["op"] == "score":
        r = rwkv7m_amd.token_logprobs(s["x"], s["tokens"], top_k=c["K"],
                                      temperature=c["temp"])
        if c["train"]:
            d, = torch.autograd.grad((r.logprobs, r.entropy), s["x"],
                                     (s["g_lp"], s["g_ent"]))
            return [r.logprobs, r.entropy, d]
        return list(r) if c["K"] else [r.logprobs, r.entropy]
    r = rwkv7m_amd.distill_loss(s["x"], s["ids"], s["top"], s["w"],
                                temperature=c["temp"])
    return [r.loss, r.row_losses, *torch.autograd.grad(r.loss, s["x"])]


def run(state):
    """One pass, as a program calls it."""
    if own:
        return _own_run(state)
    with torch.no_grad():
        return {"norm": _plain_norm, "score": _plain_score,
                "distill": _plain_distill}[state["case"]["op"]](state)


# --- what a pass cannot do without ----------------------------------------

def work(case):
    """Bytes: each input read once and each output written once.  Positions
    left out of a loss need not be read, their gradients are written."""
    c, eb = case, BYTES[case["dtype"]]
    if c["op"] == "norm":
        n, p = c["rows"] * c["C"], c["C"] * BYTES[c["ptype"]]
        if c["train"]:  # x, dy; y, dx; weight, bias and their gradients
            return {"bytes": 4 * n * eb + 4 * p, "flops": 22 * n}
        return {"bytes": 2 * n * eb + 2 * p, "flops": 8 * n}
    rows, V, K = _rows(c), c["V"], c["K"]
    if c["op"] == "score":
        if c["train"]:  # entropy is of every position
            return {"bytes": 2 * rows * V * eb + rows * 24,
                    "flops": 14 * rows * V}
        return {"bytes": rows * V * eb + rows * (16 + 12 * K),
                "flops": 8 * rows * V}
    used = rows - _left_out(c)
    return {"bytes": (used + rows) * V * eb + used * K * (8 + eb) + rows * 8,
            "flops": 10 * used * V}


# --- the definition in float64 --------------------------------------------

def _exact_norm(s):
    c = s["case"]
    w, b = s["w"].detach().double(), s["b"].detach().double()
    parts = []
    for lo in range(0, c["rows"], 4096):
        x = s["x"].detach()[lo:lo + 4096].double()
        var, mu = torch.var_mean(x, -1, correction=0, keepdim=True)
        r = 1.0 / torch.sqrt(var + 1e-5)
        n = (x - mu) * r
        part = [n * w + b]
        if c["train"]:
            dy = s["dy"][lo:lo + 4096].double()
            g = dy * w
            C = c["C"]
            part += [r / C * (C * g - g.sum(-1, keepdim=True)
                              - n * (g * n).sum(-1, keepdim=True)),
                     (dy * n).sum(0), dy.sum(0)]
        parts.append(part)
    cols = list(zip(*parts))
    out = [torch.cat(v) for v in cols[:2]]
    return out + [torch.stack(v).sum(0) for v in cols[2:]]


def _exact_score(s):
    c = s["case"]
    parts = []
    for x, tok, i in zip(s["x"].detach(), s["tokens"], range(c["B"])):
        logp = torch.log_softmax(x.double() / c["temp"], -1)
        p = torch.softmax(x.double() / c["temp"], -1)
        h = -torch.xlogy(p, p).sum(-1)
        hot = torch.zeros_like(p)
        hot.scatter_(-1, tok.clamp(min=0)[:, None], 1.0)
        hot[tok < 0] = 0.0
        part = [torch.where(hot > 0, logp, 0.0).sum(-1), h]
        if c["train"]:
            a = s["g_lp"][i].double()[:, None] * (tok >= 0)[:, None]
            e = s["g_ent"][i].double()[:, None]
            part.append((a * (hot - p) - e * (torch.xlogy(p, p)
                                              + p * h[:, None])) / c["temp"])
        elif c["K"]:
            part.append(logp.sort(-1, descending=True).values[:, :c["K"]])
        parts.append(part)
    out = [torch.stack(v) for v in zip(*parts)]
    if c["K"] and not c["train"]:
        out.insert(2, None)
    return out


def _exact_distill(s):
    c, T = s["case"], s["case"]["temp"]
    total, rows, grads = 0.0, [], []
    for x, ids, top, w in zip(s["x"].detach(), s["ids"], s["top"], s["w"]):
        w = w.double()
        q = torch.softmax((top.double() / T).masked_fill(
            ids < 0, float("-inf")), -1)
        dense = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
        dense.scatter_add_(-1, ids.clamp(min=0), q)
        lsm = torch.log_softmax(x.double() / T, -1)
        kl = (torch.xlogy(q, q).sum(-1) - (dense * lsm).sum(-1)) * T * T
        kl = kl * (w != 0)
        total = total + (w * kl).sum()
        rows.append(kl)
        grads.append(w[:, None] * T * (lsm.exp() - dense))
    return [total, torch.stack(rows), torch.stack(grads)]


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "score": _exact_score,
            "distill": _exact_distill}[case["op"]](s)

"""The operators around a language model's head (lm_norm.hip, lm_score.hip,
lm_distill.hip) against their definitions in float64.

Tolerances.  A row's sum has at most n / 64 terms in one chain (n < 2^18, so
2^12); roundings of like-signed terms average out, sqrt(2^12) 2^-24 = 4e-6
relative; SUM = 2e-5 holds that five times over.  A log probability is such a
sum's logarithm beside a difference and a product rounded at its own size:
SUM times max(1, |value|).  A gradient element is a difference of terms of
its row's coefficient (|weight| T, |d_logprobs|, ...): SUM times that.  A bf16
result is rounded once more: 2^-8 of its value.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SUM = 2e-5
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
INF = float("inf")


@pytest.fixture(scope="module")
def lm(hip_lib):
    import rwkv7m_amd
    return rwkv7m_amd


def _close(name, got, want, scale=1.0, own=True):
    """got against the float64 want: SUM * scale (or times max(scale,
    |want|) with ``own``), and 2^-8 |want| in bf16; non-finite values equal."""
    got64, want = got.detach().double().cpu(), want.detach().cpu()
    assert got64.shape == want.shape, (name, got64.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got64), fine), name
    bad = ~fine
    assert torch.equal(torch.nan_to_num(got64[bad], 0.5),
                       torch.nan_to_num(want[bad], 0.5)), name
    scale = torch.as_tensor(scale, dtype=torch.float64).cpu()
    size = torch.maximum(want.abs(), scale) if own else scale
    tol = SUM * size + (2.0 ** -8 * want.abs()
                        if got.dtype == torch.bfloat16 else 0.0)
    off = ((got64 - want).abs() - tol)[fine]
    assert not off.numel() or float(off.max()) <= 0, (name, float(off.max()))


def _gen(seed):
    return torch.Generator("cpu").manual_seed(seed)


# --- layer norm -----------------------------------------------------------

def _norm64(x, w, b, eps, dy=None):
    """(y, dx, dw, db) in float64, and the sizes their errors go by."""
    x = x.detach().double().cpu()
    C = x.shape[-1]
    w = torch.ones(C).double() if w is None else w.detach().double().cpu()
    b = torch.zeros(C).double() if b is None else b.detach().double().cpu()
    mu = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mu) * rstd
    # x - mean is off by 2^-24 of x's size
    lift = 1 + x.abs().amax(-1, keepdim=True) * rstd * 2.0 ** -6
    out = dict(y=xh * w + b, ys=lift * (w.abs() * (1 + xh.abs()) + b.abs()))
    if dy is not None:
        dy = dy.detach().double().cpu()
        g = dy * w
        out["dx"] = rstd * (g - g.mean(-1, keepdim=True)
                            - xh * (g * xh).mean(-1, keepdim=True))
        gm = g.abs().amax(-1, keepdim=True)
        out["dxs"] = lift * rstd * gm * (2 + xh.abs())
        for n, t in (("dw", dy * xh), ("db", dy), ("dbs", dy.abs()),
                     ("dws", dy.abs() * (lift + xh.abs()))):
            out[n] = t.reshape(-1, C).sum(0)
    return out


def _check_norm(lm, x, w, b, dy, eps=1e-5):
    want = _norm64(x, w, b, eps, dy)
    leaves = [t.detach().clone(memory_format=torch.preserve_format)
              if t is x else t.detach().clone()
              for t in (x, w, b) if t is not None]
    leaves[0] = x.detach().requires_grad_()
    for t in leaves[1:]:
        t.requires_grad_()
    it = iter(leaves[1:])
    wl, bl = (None if t is None else next(it) for t in (w, b))
    y = lm.layer_norm(leaves[0], wl, bl, eps)
    assert y.dtype == x.dtype
    _close("y", y, want["y"], want["ys"], own=False)
    with torch.no_grad():
        assert torch.equal(lm.layer_norm(leaves[0], wl, bl, eps), y)
    grads = torch.autograd.grad(y, leaves, dy)
    _close("dx", grads[0], want["dx"], want["dxs"], own=False)
    names = [n for n, t in (("dw", w), ("db", b)) if t is not None]
    for n, gr in zip(names, grads[1:]):
        _close(n, gr, want[n], want[n + "s"], own=False)
    again = torch.autograd.grad(lm.layer_norm(leaves[0], wl, bl, eps), leaves,
                                dy)
    assert all(torch.equal(a, c) for a, c in zip(grads, again))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("pdtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,C", [
    (1, 1), (3, 2), (5, 7), (2, 8), (1, 63), (9, 64), (4, 129), (33, 255),
    (7, 256), (700, 320), (1, 768), (517, 768), (130, 1001), (64, 2048),
    (9, 2049), (31, 4096), (5, 8191), (3, 16384), (2, 40000)])
def test_layer_norm(lm, rows, C, pdtype, dtype):
    print("case: layer norm", rows, C, dtype, pdtype, flush=True)
    g = _gen(rows * 7 + C)
    x = (torch.randn(rows, C, generator=g) * 2 + torch.randn(C, generator=g)
         ).to(DT[dtype]).cuda()
    w = (1 + 0.2 * torch.randn(C, generator=g)).to(DT[pdtype]).cuda()
    b = torch.randn(C, generator=g).to(DT[pdtype]).cuda()
    dy = torch.randn(rows, C, generator=g).to(DT[dtype]).cuda()
    _check_norm(lm, x, w, b, dy)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("with_w,with_b", [(False, False), (True, False),
                                           (False, True)])
def test_layer_norm_without_parameters(lm, with_w, with_b, dtype):
    print("case: layer norm parameters", with_w, with_b, dtype, flush=True)
    g = _gen(4)
    x = torch.randn(6, 300, generator=g).to(DT[dtype]).cuda()
    w, b = (torch.randn(300, generator=g).cuda() if on else None
            for on in (with_w, with_b))
    _check_norm(lm, x, w, b, torch.randn(6, 300, generator=g)
                .to(DT[dtype]).cuda(), eps=1e-3)


def _views(g, dtype, rows, C):
    """(name, tensor of `rows` rows of C) in layouts a program has."""
    def rnd(*s):
        return torch.randn(*s, generator=g).to(dtype).cuda()
    yield "sliced positions", rnd(rows, 5, C)[:, 1:4]
    yield "odd column offset", rnd(rows, C + 3)[:, 1:C + 1]
    yield "every other row", rnd(2 * rows, C)[::2]
    yield "three axes", rnd(rows, 3, 2, C)[:, :, 0]
    yield "swapped axes", rnd(3, rows, C).transpose(0, 1)
    yield "expanded", rnd(1, C).expand(rows, C)
    yield "columns strided", rnd(rows, C, 2)[..., 1]
    yield "one row", rnd(C)
    yield "unmergeable", rnd(2, 5, 3, C)[:, ::2, :2]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("C", [64, 771])
def test_layer_norm_layouts(lm, C, dtype):
    g = _gen(C)
    for name, x in _views(g, DT[dtype], 6, C):
        print("case: layer norm", name, C, dtype, flush=True)
        w, b = (torch.randn(C, generator=g).cuda() for _ in range(2))
        dy = torch.randn(x.shape, generator=g).to(x.dtype).cuda()
        _check_norm(lm, x, w, b, dy)
        # a cotangent that is itself broadcast (from a sum)
        xl = x.detach().requires_grad_()
        got, = torch.autograd.grad(lm.layer_norm(xl, w, b).float().sum(), xl)
        want = _norm64(x, w, b, 1e-5, torch.ones(x.shape))
        _close("dx of a sum", got, want["dx"], want["dxs"], own=False)


def test_layer_norm_hard_rows(lm):
    print("case: layer norm, constant, large, empty and non-finite rows",
          flush=True)
    C = 200
    x = torch.randn(7, C, generator=_gen(1))
    x[0] = 0.0
    x[1] = 3.0
    x[2] += 1000.0          # a mean far above the spread
    x[3] *= 1e15            # squares of 1e30
    x[4, 5] = float("nan")
    x[5, 5] = INF
    w, b = torch.ones(C), torch.zeros(C)
    y = lm.layer_norm(x.cuda(), w.cuda(), b.cuda()).cpu()
    ok = [0, 1, 2, 3, 6]
    want = _norm64(x[ok], w, b, 1e-5)
    _close("y", y[ok], want["y"], want["ys"], own=False)
    assert y[4:6].isnan().all() and not y[:2].any()
    e = torch.empty(0, C, device="cuda", requires_grad=True)
    wg = w.cuda().requires_grad_()
    junk = [torch.full((C,), float("nan"), device="cuda") for _ in range(4)]
    del junk
    out = lm.layer_norm(e, wg, None)
    out.sum().backward()
    assert out.shape == (0, C) and not wg.grad.any()


# --- token log probabilities ----------------------------------------------

def _top64(x, k):
    """Ids in the order: larger first, equal by id, NaN above +inf."""
    v = torch.where(torch.isnan(x), torch.full_like(x, INF), x)
    rank = torch.where(torch.isnan(x), 1, 0)
    out = []
    for r, row in zip(rank.reshape(-1, x.shape[-1]).tolist(),
                      v.reshape(-1, x.shape[-1]).tolist()):
        order = sorted(range(len(row)), key=lambda j: (-r[j], -row[j], j))
        out.append(order[:k])
    return torch.tensor(out, dtype=torch.int64).reshape(*x.shape[:-1], k)


def _score64(x, tok, temp):
    z = x.detach().double().cpu() / temp
    lp = torch.log_softmax(z, -1)
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    tok = tok.cpu().long()
    got = lp.gather(-1, tok.clamp(min=0)[..., None])[..., 0]
    return lp, p, ent, torch.where(tok >= 0, got, 0.0)


def _check_score(lm, x, tok, k, temp=1.0, grads=True):
    r = lm.token_logprobs(x, tok, top_k=k, temperature=temp)
    lp, p, ent, want = _score64(x, tok, temp)
    _close("logprobs", r.logprobs, want)
    _close("entropy", r.entropy, ent)
    if k:
        ids = _top64(x.float().cpu(), k)
        assert r.top_ids.dtype == torch.int64
        assert torch.equal(r.top_ids.cpu(), ids)
        _close("top", r.top_logprobs, lp.gather(-1, ids))
    else:
        assert r.top_ids is None and r.top_logprobs is None
    if not grads:
        return r
    leaf = x.detach().requires_grad_()
    q = lm.token_logprobs(leaf, tok, top_k=k, temperature=temp)
    assert torch.equal(q.logprobs, r.logprobs)
    assert torch.equal(q.entropy, r.entropy)
    g = _gen(9)
    a, e = (torch.randn(x.shape[:-1], generator=g) for _ in range(2))
    hot = torch.zeros_like(p).scatter_(
        -1, tok.cpu().long().clamp(min=0)[..., None], 1.0)
    scored = (tok.cpu() >= 0).double()[..., None]
    da = a.double()[..., None] * scored * (hot - p)
    plp = torch.where(p > 0, p * lp, 0.0)
    de = -e.double()[..., None] * (plp + p * ent[..., None])
    scale = (a.abs() + e.abs() * (1 + ent.abs()))[..., None].double() / temp
    for name, out, cot, d in (
            ("both", (q.logprobs, q.entropy), (a, e), da + de),
            ("logprobs", (q.logprobs,), (a,), da),
            ("entropy", (q.entropy,), (e,), de)):
        got, = torch.autograd.grad(out, leaf, [c.cuda() for c in cot],
                                   retain_graph=True)
        assert got.dtype == x.dtype
        _close("gradient of " + name, got, d / temp, scale, own=False)
    return r


def _logits(g, *shape, dtype="bf16"):
    return (3 * torch.randn(*shape, generator=g)).to(DT[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,V,k,temp", [
    (1, 1, 1, 1.0), (3, 2, 2, 1.0), (2, 7, 7, 0.5), (4, 8, 3, 1.0),
    (5, 9, 0, 2.0), (2, 63, 63, 1.0), (3, 64, 64, 1.0), (2, 65, 64, 0.7),
    (70, 257, 5, 1.0), (3, 1000, 64, 1.0), (2, 2049, 33, 1.3),
    (5, 4103, 20, 1.0), (1, 32003, 64, 0.7), (2, 65536, 20, 1.0),
    (1, 131073, 40, 1.0), (600, 300, 1, 1.0)])
def test_token_logprobs(lm, rows, V, k, temp, dtype):
    print("case: token logprobs", rows, V, k, temp, dtype, flush=True)
    g = _gen(rows + V)
    x = _logits(g, rows, V, dtype=dtype).cuda()
    tok = torch.randint(0, V, (rows,), generator=g)
    tok[rows // 2] = -100 if rows > 1 else tok[0]
    _check_score(lm, x, tok.cuda(), k, temp)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [64, 1009])
def test_token_logprobs_layouts(lm, V, dtype):
    g = _gen(V)
    for name, x in _views(g, DT[dtype], 6, V):
        print("case: token logprobs", name, V, dtype, flush=True)
        tok = torch.randint(0, V, x.shape[:-1], generator=g).to(torch.int32)
        _check_score(lm, x, tok.cuda(), 4)


def _rows_like(kind, V, dtype):
    """Rows whose largest logits lie where a selection could go wrong."""
    x = _logits(_gen(3), 1, V, dtype=dtype)[0]
    i = torch.arange(V)
    if kind == "equal":
        x[:] = 1.5
    elif kind == "zeros of both signs":
        x[:] = torch.where(i % 3 == 0, -0.0, 0.0).to(x.dtype)
    elif kind == "rising":
        x[:] = (i.float() / V * 8).to(x.dtype)
    elif kind == "falling":
        x[:] = (-i.float() / V * 8).to(x.dtype)
    elif kind == "two values":
        x[:] = torch.where(i % 2 == 0, 1.0, 2.0).to(x.dtype)
    elif kind == "one block of large ones":
        x[V // 3:V // 3 + V // 8] += 20
    elif kind.startswith("stride "):
        x[::int(kind.split()[1])] += 20
    elif kind == "ties at the edge":
        x[:] = -1.0
        x[V // 2:] = 0.0
        x[V - 3:] = 1.0
    elif kind == "negative":
        x[:] = -x.abs() - 50
    return x


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [1000, 20011, 65536])
def test_top_alternatives_of_hard_rows(lm, V, dtype):
    kinds = ["equal", "zeros of both signs", "rising", "falling",
             "two values", "one block of large ones", "ties at the edge",
             "negative", "stride 8", "stride 64", "stride 256", "stride 512",
             "stride 2048", "stride 4096", "stride 8192"]
    x = torch.stack([_rows_like(kd, V, dtype) for kd in kinds]).cuda()
    tok = torch.zeros(len(kinds), dtype=torch.int64, device="cuda")
    for k in (1, 20, 64):
        print("case: hard rows", V, k, dtype, flush=True)
        _check_score(lm, x, tok, k, grads=k == 1)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [40, 5000])
def test_token_logprobs_masked_rows(lm, V, dtype):
    """-inf masks up to all of a row, the type's lowest and largest values."""
    print("case: masked rows", V, dtype, flush=True)
    g = _gen(V)
    x = _logits(g, 7, V, dtype=dtype)
    x[0, torch.rand(V, generator=g) < 0.5] = -INF
    x[1] = -INF
    x[1, V - 2] = 2.0                      # one allowed
    x[2] = torch.finfo(DT[dtype]).min      # uniform
    x[3, 5:] = torch.finfo(DT[dtype]).min
    x[4] = torch.finfo(DT[dtype]).max      # uniform
    x[5, 1::2] = -INF
    x[6] = 0.0
    tok = torch.tensor([3, V - 2, 1, 2, 0, 1, 0]).cuda()
    _check_score(lm, x.cuda(), tok, min(20, V))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_token_logprobs_rows_without_a_distribution(lm, dtype):
    print("case: empty, NaN and +inf rows", dtype, flush=True)
    V, k = 3000, 9
    x = _logits(_gen(1), 6, V, dtype=dtype)
    x[0] = -INF
    x[1, 77] = float("nan")
    x[2, 5] = INF
    x[3] = float("nan")
    x[4, 9], x[4, 4] = float("nan"), INF
    tok = torch.tensor([4, 3, 2, 1, 0, V + 5]).cuda()
    leaf = x.cuda().requires_grad_()
    r = lm.token_logprobs(leaf, tok, top_k=k)
    assert r.logprobs[0] == -INF and r.entropy[0] == 0
    assert (r.top_logprobs[0] == -INF).all()
    assert r.logprobs[1:].isnan().all() and r.entropy[1:5].isnan().all()
    assert r.top_logprobs[1:5].isnan().all()
    assert torch.isfinite(r.entropy[5]) and r.top_logprobs[5].isfinite().all()
    assert torch.equal(r.top_ids.cpu(), _top64(x.float(), k))
    # the gradient: p = 0 in the empty row; rows left out by their cotangent
    cot = torch.tensor([2.0, 0, 0, 0, 0, 0]).cuda()
    d, = torch.autograd.grad(r.logprobs, leaf, cot, retain_graph=True)
    want = torch.zeros(6, V)
    want[0, 4] = 2.0
    assert torch.equal(d.float().cpu(), want)
    d, = torch.autograd.grad(r.logprobs, leaf, torch.ones(6).cuda())
    assert d[1:].isnan().all() and torch.isfinite(d[0]).all()


# --- distillation ---------------------------------------------------------

def _distill64(x, ids, top, w, T):
    x, top = x.detach().double().cpu(), top.double().cpu()
    ids = ids.cpu().long()
    rows = x.shape[:-1].numel()
    w = torch.full(x.shape[:-1], 1.0 / max(1, rows), dtype=torch.float64) \
        if w is None else w.double().cpu()
    t = (top / T).masked_fill(ids < 0, -INF)
    used = (w != 0) & (t.amax(-1) != -INF) if t.shape[-1] else w < -INF
    logq = torch.log_softmax(t, -1)
    q = torch.where(used[..., None], logq.exp(), 0.0)
    lsm = torch.log_softmax(x / T, -1)
    term = q * (logq - lsm.gather(-1, ids.clamp(min=0)))
    kl = T * T * torch.where(q > 0, term, 0.0).sum(-1)
    dense = torch.zeros_like(x).scatter_add_(-1, ids.clamp(min=0), q)
    d = torch.where(used[..., None], (w * T)[..., None] * (lsm.exp() - dense),
                    0.0)
    return torch.where(used, w * kl, 0.0).sum(), kl, d, (w.abs() * T)[..., None]


def _check_distill(lm, x, ids, top, w, T):
    leaf = x.detach().requires_grad_()
    r = lm.distill_loss(leaf, ids, top, w, temperature=T)
    loss, rows, d, scale = _distill64(x, ids, top, w, T)
    size = T * T * max(1.0, float(rows.abs().max())) if rows.numel() else 1.0
    _close("row losses", r.row_losses, rows, size)
    total = float(scale.sum()) / T if rows.numel() else 1.0
    _close("loss", r.loss, loss, size * max(total, 1e-30), own=False)
    assert not r.row_losses.requires_grad
    with torch.no_grad():
        again = lm.distill_loss(leaf, ids, top, w, temperature=T)
    assert torch.equal(again.loss, r.loss)
    assert torch.equal(again.row_losses, r.row_losses)
    got, = torch.autograd.grad(r.loss, leaf, retain_graph=True)
    assert got.dtype == x.dtype
    _close("gradient", got, d, scale, own=False)
    # over the retained graph once more, and scaled
    second, = torch.autograd.grad(r.loss, leaf, retain_graph=True)
    assert torch.equal(second, got) and (not got.numel() or
                                         second.data_ptr() != got.data_ptr())
    scaled, = torch.autograd.grad(3.0 * r.loss, leaf)
    _close("scaled gradient", scaled, 3.0 * d, 3.0 * scale, own=False)
    first = lm.distill_loss(leaf, ids, top, w, temperature=T).loss * -0.5
    scaled, = torch.autograd.grad(first, leaf)
    _close("scaled gradient", scaled, -0.5 * d, scale, own=False)


def _teacher(g, shape, V, K, dtype="f32"):
    flat = [torch.randperm(V, generator=g)[:K] for _ in range(shape.numel())]
    ids = (torch.stack(flat) if flat else torch.zeros(0, K).long()).reshape(
        *shape, K)
    return ids, (3 * torch.randn(*shape, K, generator=g)).to(DT[dtype])


@pytest.mark.parametrize("dtype,tdtype", [("bf16", "bf16"), ("bf16", "f32"),
                                          ("f32", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("rows,V,K,T", [
    (1, 1, 1, 1.0), (3, 2, 2, 2.0), (2, 9, 9, 1.0), (5, 64, 16, 0.5),
    (70, 257, 3, 1.0), (4, 1003, 256, 1.5), (2, 4096, 64, 1.0),
    (3, 8200, 100, 2.0), (2, 32003, 50, 1.0), (2, 65536, 64, 2.0),
    (1, 65529, 7, 1.0), (2, 131072, 16, 1.0), (1, 150001, 8, 1.0),
    (1, 270003, 8, 1.0)])
def test_distill_loss(lm, rows, V, K, T, dtype, tdtype):
    print("case: distill", rows, V, K, T, dtype, tdtype, flush=True)
    g = _gen(rows + V + K)
    x = _logits(g, rows, V, dtype=dtype).cuda()
    ids, top = _teacher(g, torch.Size((rows,)), V, K, tdtype)
    w = torch.rand(rows, generator=g) + 0.1
    _check_distill(lm, x, ids.cuda(), top.cuda(), w.cuda(), T)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [64, 1009])
def test_distill_layouts(lm, V, dtype):
    g = _gen(V)
    for name, x in _views(g, DT[dtype], 6, V):
        print("case: distill", name, V, dtype, flush=True)
        ids, top = _teacher(g, x.shape[:-1], V, 5)
        _check_distill(lm, x, ids.to(torch.int32).cuda(), top.cuda(), None,
                       1.0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V,K", [(50, 6), (9001, 200)])
def test_distill_ragged_teachers(lm, V, K, dtype):
    """Absent, masked, repeated and unordered alternatives, rows left out."""
    print("case: distill ragged", V, K, dtype, flush=True)
    g = _gen(V)
    x = _logits(g, 8, V, dtype=dtype)
    ids, top = _teacher(g, torch.Size((8,)), V, min(K, V))
    K = ids.shape[-1]
    w = torch.rand(8, generator=g) + 0.5
    ids[0, K // 2:] = -1
    ids[1] = -1                       # no alternative
    top[2, ::2] = -INF
    top[3] = -INF                     # no alternative above -inf
    ids[4] = ids[4, 0]                # one id K times
    ids[5, 1::2] = ids[5, 0]
    w[6] = 0.0
    x[6] = float("nan")               # left out, whatever it holds
    top[6], ids[6] = float("nan"), V + 1
    x[1, 3] = INF
    leaf = x.cuda().requires_grad_()
    r = lm.distill_loss(leaf, ids.cuda(), top.cuda(), w.cuda())
    d, = torch.autograd.grad(r.loss, leaf)
    assert not d[[1, 3, 6]].any() and not r.row_losses[[1, 3, 6]].any()
    keep = [0, 2, 4, 5, 7]
    loss, rows, want, scale = _distill64(x[keep], ids[keep], top[keep],
                                         w[keep], 1.0)
    _close("rows", r.row_losses[keep], rows)
    _close("loss", r.loss, loss, float(rows.abs().max()) * float(w.sum()),
           own=False)
    _close("gradient", d[keep], want, scale, own=False)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_distill_rows_without_a_distribution(lm, dtype):
    print("case: distill, masked and non-finite students", dtype, flush=True)
    V = 700
    x = _logits(_gen(2), 6, V, dtype=dtype)
    ids, top = _teacher(_gen(3), torch.Size((6,)), V, 4)
    x[0] = -INF                              # p = 0: infinite loss
    x[1, ids[1, 0]] = -INF                   # one of the teacher's masked
    x[2, 9] = float("nan")
    x[3] = torch.finfo(DT[dtype]).min        # uniform
    ids[4, 2] = V                            # beyond the vocabulary
    x[5, :] = -INF
    x[5, ids[5]] = 1.0                       # nothing but the teacher's
    leaf = x.cuda().requires_grad_()
    w = torch.ones(6)
    r = lm.distill_loss(leaf, ids.cuda(), top.cuda(), w.cuda())
    d, = torch.autograd.grad(r.loss, leaf)
    d = d.double().cpu()
    assert r.row_losses[0] == INF and r.row_losses[1] == INF
    assert r.row_losses[2].isnan() and r.row_losses[4].isnan()
    assert r.loss.isnan()
    assert d[2].isnan().all() and d[4].isnan().all()
    ok = [3, 5]
    _, rows, want, scale = _distill64(x[ok], ids[ok], top[ok], w[ok], 1.0)
    _close("rows", r.row_losses[ok].cpu(), rows)
    got = torch.as_tensor(d[ok]).to(DT[dtype])
    _close("gradient", got, want, scale, own=False)
    q = torch.softmax(top.double(), -1)
    for i in (0, 1):
        base = torch.softmax(x[i].double(), -1) if i else torch.zeros(V)
        want = base.double().scatter_add(0, ids[i], -q[i])
        _close("gradient", d[i].to(DT[dtype]), want, own=False)


def test_distill_without_rows_or_alternatives(lm):
    print("case: distill, nothing to do", flush=True)
    junk = [torch.full((n,), float("nan"), device="cuda")
            for n in (1, 3, 60) for _ in range(4)]
    del junk
    x = torch.randn(3, 20, device="cuda", requires_grad=True)
    r = lm.distill_loss(x, torch.zeros(3, 0, dtype=torch.int64).cuda(),
                        torch.zeros(3, 0).cuda())
    assert r.loss == 0 and not r.row_losses.any()
    assert not torch.autograd.grad(r.loss, x)[0].any()
    e = torch.randn(2, 0, 20, device="cuda", requires_grad=True)
    r = lm.distill_loss(e, torch.zeros(2, 0, 4, dtype=torch.int64).cuda(),
                        torch.zeros(2, 0, 4).cuda())
    assert r.loss == 0 and torch.autograd.grad(r.loss, e)[0].shape == e.shape
    s = lm.token_logprobs(e, torch.zeros(2, 0, dtype=torch.int64).cuda(),
                          top_k=2)
    assert s.top_ids.shape == (2, 0, 2) and s.logprobs.shape == (2, 0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [9, 2047, 2051, 8203, 16387, 20005, 32769,
                               40003, 65531, 131075, 140007])
def test_every_place_of_a_row_counts(lm, V, dtype):
    """Rows with all their weight at their ends or in the middle: each element
    there is most of the sum, of the gradient and of the alternatives."""
    print("case: weight at the ends", V, dtype, flush=True)
    x = _logits(_gen(V), 4, V, dtype=dtype)
    ends = list(range(min(V, 12))) + list(range(max(0, V - 12), V))
    x[0, ends] = 20.0 + torch.arange(float(len(ends))).to(x.dtype) / 8
    x[1, V - 1] = 30.0
    x[2, :] = -INF
    x[2, ends[::2]] = 1.0
    x[3, V // 2 - 1:V // 2 + 9] = 25.0
    tok = torch.tensor([V - 1, V - 1, ends[0], V // 2]).cuda()
    _check_score(lm, x.cuda(), tok, min(V, 30))
    ids = torch.tensor([[V - 1, 0], [V - 2, V - 1], [ends[0], ends[2]],
                        [V // 2, V - 1]]).cuda()
    top = torch.tensor([[1.0, 2.0], [0.5, 0.0], [0.0, 0.0], [3.0, 1.0]]).cuda()
    _check_distill(lm, x.cuda(), ids, top, None, 1.0)


# --- gradients against differences ----------------------------------------

def _against_differences(f, leaves, step=1e-2):
    """The gradient along a random direction against the central difference:
    truncation step^2 / 6 of a third derivative of order one, rounding 2^-24
    of the value over the step: 1e-3 of the direction's size."""
    g = _gen(11)
    dirs = [torch.randn(t.shape, generator=g).cuda() for t in leaves]
    grads = torch.autograd.grad(f(*leaves), leaves)
    got = sum(float((a.double() * b.double()).sum())
              for a, b in zip(grads, dirs))
    with torch.no_grad():
        hi, lo = (float(f(*(t + s * step * d for t, d in zip(leaves, dirs))))
                  for s in (1, -1))
    want = (hi - lo) / (2 * step)
    size = math.sqrt(sum(float(a.double().square().sum()) for a in grads))
    assert size > 0 and abs(got - want) <= 1e-3 * max(1.0, size) + \
        2e-2 * step * max(1.0, abs(hi)), (got, want)


def test_gradients_against_differences(lm):
    print("case: gradients against differences", flush=True)
    g = _gen(5)

    def leaf(*s):
        return torch.randn(*s, generator=g).cuda().requires_grad_()

    cot = torch.randn(5, 33, generator=g).cuda()
    _against_differences(lambda x, w, b: (lm.layer_norm(x, w, b) * cot).sum(),
                         [leaf(5, 33), leaf(33), leaf(33)])
    tok = torch.tensor([3, -1, 30, 7], device="cuda")
    c1, c2 = (torch.randn(4, generator=g).cuda() for _ in range(2))

    def score(x):
        r = lm.token_logprobs(x, tok, temperature=1.3)
        return (r.logprobs * c1).sum() + (r.entropy * c2).sum()

    _against_differences(score, [leaf(4, 33)])
    ids, top = _teacher(g, torch.Size((4,)), 33, 6)
    _against_differences(
        lambda x: lm.distill_loss(x, ids.cuda(), top.cuda(),
                                  temperature=1.7).loss, [leaf(4, 33)])


def test_second_derivatives_are_refused(lm):
    print("case: second derivatives", flush=True)
    x = torch.randn(2, 16, device="cuda", requires_grad=True)
    for out in (lm.layer_norm(x).square().sum(),
                lm.token_logprobs(x, torch.zeros(2, dtype=torch.int64,
                                                 device="cuda")).entropy.sum(),
                lm.distill_loss(x, torch.zeros(2, 1, dtype=torch.int64,
                                               device="cuda"),
                                torch.zeros(2, 1, device="cuda")).loss):
        d, = torch.autograd.grad(out, x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable|does not "
                                               "require grad"):
            d.sum().backward()


# --- large offsets, streams, graphs ---------------------------------------

def test_offsets_past_32_bits(lm):
    """Rows more than 2^32 bytes into the logits, and the same in the
    gradient and in a norm: equal to the same rows alone, bit for bit."""
    print("case: offsets past 32 bits", flush=True)
    rows, V = 34000, 65536
    big = torch.zeros(rows, V, dtype=torch.bfloat16, device="cuda")
    last = 3 * torch.randn(3, V, generator=_gen(8)).to(torch.bfloat16).cuda()
    big[-3:] = last
    ids = torch.arange(rows * 4, device="cuda").view(rows, 4) % V
    top = torch.randn(rows, 4, generator=_gen(9)).cuda()
    w = torch.zeros(rows, device="cuda")
    w[-3:] = torch.tensor([1.0, 2.0, 0.5])
    x, y = big.requires_grad_(), last.clone().requires_grad_()
    a = lm.distill_loss(x, ids, top, w)
    b = lm.distill_loss(y, ids[-3:], top[-3:], w[-3:])
    assert torch.equal(a.row_losses[-3:], b.row_losses)
    da, = torch.autograd.grad(a.loss, x)
    db, = torch.autograd.grad(b.loss, y)
    assert torch.equal(da[-3:], db)
    del da, db, a, b
    tok = ids[:, 0].contiguous()
    cot = torch.zeros(rows, device="cuda")
    cot[-3:] = 1.0
    a = lm.token_logprobs(x, tok, top_k=3)
    b = lm.token_logprobs(y, tok[-3:], top_k=3)
    assert all(torch.equal(p[-3:], q) for p, q in zip(a, b))
    da, = torch.autograd.grad(a.logprobs, x, cot)
    db, = torch.autograd.grad(b.logprobs, y, cot[-3:])
    assert torch.equal(da[-3:], db)
    del da, db, a, b
    # two rows 2^31 + 5 elements apart, and a norm's output past 2^32 bytes
    far = big.detach().view(-1).as_strided((2, 1000), (2 ** 31 + 5, 1))
    near = far.contiguous()
    assert torch.equal(lm.layer_norm(far), lm.layer_norm(near))
    assert torch.equal(lm.token_logprobs(far, tok[:2]).entropy,
                       lm.token_logprobs(near, tok[:2]).entropy)
    out = lm.layer_norm(big.detach())
    assert torch.equal(out[-3:], lm.layer_norm(last))


def _all_ops(lm, x, w, tok, ids, top):
    leaves = [x, w]
    h = lm.layer_norm(x, w)
    s = lm.token_logprobs(h, tok, top_k=4)
    r = lm.distill_loss(h, ids, top)
    g = torch.autograd.grad(
        (r.loss, s.logprobs, s.entropy), leaves,
        (torch.full_like(r.loss, 2.0), torch.ones_like(s.logprobs),
         torch.ones_like(s.entropy)))
    return [h.detach(), *(t.detach() for t in s), r.loss.detach(),
            r.row_losses, *g]


def _all_inputs(seed):
    g = _gen(seed)
    x = torch.randn(40, 2000, generator=g).to(torch.bfloat16).cuda()
    w = (1 + torch.rand(2000, generator=g)).cuda()
    ids, top = _teacher(g, torch.Size((40,)), 2000, 8)
    tok = torch.randint(0, 2000, (40,), generator=g)
    return [x.requires_grad_(), w.requires_grad_(), tok.cuda(), ids.cuda(),
            top.cuda()]


def test_side_stream_and_graph_replays(lm):
    print("case: side stream, then a graph replayed", flush=True)
    args, other = _all_inputs(1), _all_inputs(2)
    want = _all_ops(lm, *args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _all_ops(lm, *args)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.cuda.stream(side):
        _all_ops(lm, *args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = _all_ops(lm, *args)
    for rep in range(3):
        for t in out:
            t.fill_(-7)
        _all_ops(lm, *other)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), f"replay {rep}"


# --- more rows than a grid's columns, parts of the gradients, the example ---

def test_more_rows_than_65536(lm):
    print("case: 70001 rows", flush=True)
    rows, V = 70001, 10
    x = torch.randn(rows, V, generator=_gen(1)).cuda()
    last = x[-3:].clone()
    tok = torch.arange(rows, device="cuda") % V
    a = lm.token_logprobs(x, tok, top_k=3)
    b = lm.token_logprobs(last, tok[-3:], top_k=3)
    assert all(torch.equal(p[-3:], q) for p, q in zip(a, b))
    ids, top = tok[:, None].contiguous(), torch.zeros(rows, 1, device="cuda")
    w = torch.ones(rows, device="cuda")
    a = lm.distill_loss(x, ids, top, w)
    b = lm.distill_loss(last, ids[-3:], top[-3:], w[-3:])
    assert torch.equal(a.row_losses[-3:], b.row_losses)
    want = a.row_losses.double().sum()
    assert abs(float(a.loss.double() - want)) <= 1e-6 * float(want)
    assert torch.equal(lm.layer_norm(x)[-3:], lm.layer_norm(last))


@pytest.mark.parametrize("C", [100, 3000, 20000])
def test_layer_norm_gradients_one_at_a_time(lm, C):
    """Each of the three gradients alone is that of all three together."""
    print("case: layer norm, parts of the gradients", C, flush=True)
    g = _gen(C)
    x, w, b = (torch.randn(*s, generator=g).cuda() for s in
               ((9, C), (C,), (C,)))
    dy = torch.randn(9, C, generator=g).cuda()
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    every = torch.autograd.grad(lm.layer_norm(*leaves), leaves, dy)
    for i in range(3):
        args = [x, w, b]
        args[i] = leaves[i]
        got, = torch.autograd.grad(lm.layer_norm(*args), leaves[i], dy)
        assert torch.equal(got, every[i])
    got, = torch.autograd.grad(lm.layer_norm(x, None, leaves[2]), leaves[2],
                               dy)
    assert torch.equal(got, every[2])


def test_the_example_learns(hip_lib):
    print("case: distill and score example", flush=True)
    import importlib.util
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    spec = importlib.util.spec_from_file_location(
        "distill_and_score",
        os.path.join(root, "examples", "distill_and_score.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    losses, before, after = mod.run(steps=25, vocab=5003, width=256)
    assert torch.isfinite(losses).all()
    assert float(losses[-1]) < 0.7 * float(losses[0])
    assert float(after.logprobs.mean()) > float(before.logprobs.mean())
    assert after.top_ids.shape == (4, 64, 3)


# --- the softmax over every temperature and size of logit that is accepted --

def _check_distill_range(lm, x, ids, top, w, T):
    """As _check_distill, with the row losses' tolerance by their terms: q_k
    is off by SUM of itself, log q_k and log p_k by SUM times max(1, |value|),
    and what fp32 cannot hold (2^-149) is 0."""
    leaf = x.cuda().requires_grad_()
    r = lm.distill_loss(leaf, ids.cuda(), top.cuda(), w.cuda(), temperature=T)
    d, = torch.autograd.grad(r.loss, leaf, retain_graph=True)
    scaled, = torch.autograd.grad(-2.0 * r.loss, leaf)
    loss, rows, want, scale = _distill64(x, ids, top, w, T)
    logq = torch.log_softmax((top.double() / T).masked_fill(ids < 0, -INF), -1)
    lp = torch.log_softmax(x.double() / T, -1).gather(-1, ids.clamp(min=0))
    q = logq.exp()
    size = sum(torch.where(q > 0, q * v.abs().clamp(min=1.0), 0.0).sum(-1)
               for v in (logq, lp))
    tol = 2 * SUM * T * T * size + 2.0 ** -149
    off = (r.row_losses.double().cpu() - rows).abs()
    assert bool((off <= tol).all()), (T, off, tol)
    off = abs(float(r.loss) - float(loss))
    assert off <= float((w.double() * tol).sum()) + 1e-7 * abs(float(loss)), (
        T, off)
    _close("gradient", d, want, scale, own=False)
    _close("scaled gradient", scaled, -2 * want, 2 * scale, own=False)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [300, 5000, 40003])
def test_softmax_at_every_temperature(lm, V, dtype):
    """Down to greedy: the exponents go up to 1e32, past fp32's whole
    numbers."""
    g = _gen(V)
    x = _logits(g, 6, V, dtype=dtype).clamp(max=19.0)
    x[0, 7] = 30.25
    x[1, V - 2] = 23.5
    x[2, [3, V // 2, V - 1]] = 30.25       # three of the same
    x[3, 11] = 20.0
    x[4] = -x[4].abs() - 2.5               # the largest is negative
    x[5, ::2] = -INF
    tok = torch.tensor([7, V - 2, 3, 12, 0, 1])
    ids, top = _teacher(g, torch.Size((6,)), V, 9)
    ids[:, 0] = x.float().argmax(-1)
    ids[5] = 1 + 2 * torch.arange(9)       # none of the masked
    top[0, 3], top[1, 0], top[2, 1:3] = 30.25, 23.5, 20.0
    w = torch.rand(6, generator=g) + 0.5
    for e in (3, 1, *range(-3, -31, -1)):
        T = 10.0 ** e
        print("case: temperature", V, dtype, T, flush=True)
        _check_score(lm, x.cuda(), tok.cuda(), 3 if V == 300 else 0, T)
        _check_distill_range(lm, x, ids, top, w, T)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [300, 5000, 40003])
def test_softmax_at_every_size_of_logits(lm, V, dtype):
    """Rows of one value throughout (a mask's), a few beside it, and rows that
    spread around it, student and teacher."""
    g = _gen(V + 1)
    for e in (3, 4, 5, 6, 7, 8, 9, 10, 12, 16, 20, 25, 29, 30, 31, 38):
        print("case: size of logits", V, dtype, e, flush=True)
        at = torch.tensor([-1.0, 1.0, -1.0, 1.0, -1.0, 1.0]) * 10.0 ** e
        x = at[:, None].expand(6, V).clone()
        x[2:4] += 3 * torch.randn(2, V, generator=g)
        x[4:] *= 1 + 2.0 ** -7 * torch.rand(2, V, generator=g)
        x[1, V // 3] *= 1.0 + 2.0 ** -6
        x = x.to(DT[dtype])
        ids, top = _teacher(g, torch.Size((6,)), V, 9)
        top = top + (at * torch.tensor([1.0, 0, 1, 0, 0, -1]))[:, None]
        top[0], top[1, :5] = at[0], -10.0 ** e
        tok = ids[:, 0].clone()
        w = torch.rand(6, generator=g) + 0.5
        _check_score(lm, x.cuda(), tok.cuda(), 3 if V == 300 else 0)
        _check_distill_range(lm, x, ids, top, w, 1.0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_results_that_fit_where_a_difference_does_not(lm, dtype):
    """x - largest, or the loss before T^2, past fp32's range: the log
    probability at a high temperature and the loss at a low one are within."""
    V = 300
    g = _gen(21)
    x = _logits(g, 4, V, dtype="f32")
    x[0, ::3], x[0, 1::3] = -3e38, 3e38
    x[1] = -3.2e38
    x[1, 5] = 3.2e38
    x[2, 4], x[2, 9] = 1e30, -1e30
    x[3, :9] *= 1e12
    x = x.to(DT[dtype])
    tok = torch.tensor([0, 0, 9, 3])
    for T in (2.0, 3.7, 1e4, 1e20, 1e30):
        print("case: differences past fp32, scored", dtype, T, flush=True)
        _check_score(lm, x.cuda(), tok.cuda(), 64, T)
    # the teacher sure of what the student all but excludes
    ids = torch.tensor([[0, 1, 2], [0, 5, 7], [9, 4, 3], [3, 8, 100]])
    top = torch.tensor([[3.0, 1.0, 0.0], [3e38, -3e38, -3e38],
                        [1e30, -1e30, 0.0], [1e12, 0.0, 1e11]])
    w = torch.rand(4, generator=g) + 0.5
    for T in (0.1, 1e-3, 1e-8, 1e-30):
        print("case: differences past fp32, distilled", dtype, T, flush=True)
        _check_distill_range(lm, x, ids, top, w, T)


# --- what a row's bits depend on ------------------------------------------

def _placed(row, past, dtype):
    """A copy of the row whose address is `past` elements above a multiple of
    16 bytes."""
    buf = torch.zeros(row.numel() + 64, dtype=dtype, device="cuda")
    first = -buf.data_ptr() % 16 // buf.element_size()
    out = buf[first + past:first + past + row.numel()]
    assert out.data_ptr() % 16 == past * buf.element_size()
    return out.copy_(row)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [61, 1001, 5003, 20011, 65529, 140007])
def test_bits_of_a_row_by_its_alignment(lm, V, dtype):
    """The rows of a batch of odd length against each alone: equal bits at
    the same address modulo 16, else equal ids and values to rounding."""
    print("case: alignment of rows", V, dtype, flush=True)
    g = _gen(V)
    dt = DT[dtype]
    n = 16 // torch.empty((), dtype=dt).element_size()
    x = _logits(g, n + 1, V, dtype=dtype).cuda()
    assert x.data_ptr() % 16 == 0
    tok = torch.randint(0, V, (n + 1,), generator=g).cuda()
    ids, top = (t.cuda() for t in _teacher(g, torch.Size((n + 1,)), V, 5))
    w = torch.ones(n + 1, device="cuda")

    def scored(x, s):
        x = x.detach().requires_grad_()
        r = lm.token_logprobs(x, tok[s], top_k=5)
        d, = torch.autograd.grad((r.logprobs.sum(), r.entropy.sum()), x)
        k = lm.distill_loss(x, ids[s], top[s], w[s])
        dk, = torch.autograd.grad(k.loss, x)
        return [*r, k.row_losses, d, dk]

    every = scored(x, slice(None))
    for r in (0, 1, n // 2, n - 1, n):
        s, past = slice(r, r + 1), r * V % n
        same = scored(_placed(x[r], past, dt)[None], s)
        for a, b in zip(every, same):
            assert torch.equal(a[s], b)
        other = scored(_placed(x[r], (past + 1) % n, dt)[None], s)
        assert torch.equal(every[2][s], other[2])
        for i in (0, 1, 3, 4):
            _close("value", other[i], every[i][s].double())
        for i in (5, 6):  # (two roundings to bf16 may fall a step apart)
            a, b = other[i].double(), every[i][s].double()
            step = 2.0 ** -7 * b.abs() if dtype == "bf16" else 0.0
            assert bool(((a - b).abs() <= 14 * SUM + step).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [500, 2048, 20000])
def test_bits_of_a_row_by_its_alternatives(lm, V, dtype):
    """Equal for 0 to 40 alternatives and 0 to 64 of the teacher's, for any
    number in rows of more than 512 vectors of 16 bytes."""
    print("case: number of alternatives", V, dtype, flush=True)
    g = _gen(V)
    x = _logits(g, 3, V, dtype=dtype).cuda()
    tok = torch.randint(0, V, (3,), generator=g).cuda()
    ids, top = (t.cuda() for t in _teacher(g, torch.Size((3,)), V, 4))
    long = V * x.element_size() > 512 * 16
    base = lm.token_logprobs(x, tok)
    for k in (1, 5, 40, 41, 64):
        r = lm.token_logprobs(x, tok, top_k=k)
        if k <= 40 or long:
            assert torch.equal(r.logprobs, base.logprobs)
            assert torch.equal(r.entropy, base.entropy)
        else:
            _close("logprobs", r.logprobs, base.logprobs.double())
            _close("entropy", r.entropy, base.entropy.double())
    base = lm.distill_loss(x, ids, top).row_losses
    for k in (5, 64, 65, 256):
        more = torch.full((3, k - 4), -1, device="cuda")
        got = lm.distill_loss(
            x, torch.cat([ids, more], -1),
            torch.cat([top, more.float()], -1)).row_losses
        if k <= 64 or long:
            assert torch.equal(got, base)
        else:
            _close("row losses", got, base.double())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_unscored_tokens_of_rows_without_a_distribution(lm, dtype):
    """A token below 0 has logprob 0 whatever its row holds; the entropy and
    the alternatives are the row's."""
    print("case: unscored tokens of NaN rows", dtype, flush=True)
    V = 900
    x = _logits(_gen(6), 4, V, dtype=dtype)
    x[0, 5], x[1, 6], x[2] = float("nan"), INF, -INF
    tok = torch.full((4,), -100).cuda()
    leaf = x.cuda().requires_grad_()
    r = lm.token_logprobs(leaf, tok, top_k=3)
    assert not r.logprobs.any() and r.entropy[:2].isnan().all()
    assert r.entropy[2] == 0 and r.top_logprobs[:2].isnan().all()
    assert torch.equal(r.top_ids.cpu(), _top64(x.float(), 3))
    d, = torch.autograd.grad(r.logprobs, leaf, torch.ones(4).cuda())
    assert not d.any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_distill_non_finite_teachers_and_students(lm, dtype):
    print("case: distill, NaN and +inf on either side", dtype, flush=True)
    V = 900
    x = _logits(_gen(7), 5, V, dtype=dtype)
    ids, top = _teacher(_gen(8), torch.Size((5,)), V, 6)
    x[0, 5], x[1, 6] = INF, float("nan")
    top[2, 1], top[3, 4] = INF, float("nan")
    top[4, 3], ids[4, 3] = float("nan"), -1     # absent: not looked at
    leaf = x.cuda().requires_grad_()
    r = lm.distill_loss(leaf, ids.cuda(), top.cuda())
    d, = torch.autograd.grad(r.loss, leaf)
    assert r.row_losses[:4].isnan().all() and r.row_losses[4].isfinite()
    assert d[:2].isnan().all() and d[4].isfinite().all()
    at = torch.zeros(2, V, dtype=torch.bool).scatter_(1, ids[2:4], True)
    assert torch.equal(d[2:4].isnan().cpu(), at)


# --- gradients where a workgroup takes more than one turn -------------------

@pytest.mark.parametrize("dtype,rows,C", [
    ("bf16", 40001, 40), ("f32", 40001, 40),       # 16 threads a row
    ("bf16", 9001, 320), ("f32", 9001, 500),       # a wave, one and two vectors
    ("bf16", 9001, 1000),
    ("bf16", 2731, 1536), ("f32", 2731, 1001),     # 4 waves
    ("bf16", 2600, 4096), ("f32", 2600, 2048),
    ("bf16", 600, 8191), ("f32", 600, 4093),       # 16 waves
    ("bf16", 517, 16384), ("f32", 517, 8192),
    ("bf16", 600, 5), ("f32", 600, 3),             # element by element
    ("bf16", 300, 20000), ("f32", 300, 20000)])
def test_layer_norm_gradients_of_many_rows(lm, dtype, rows, C):
    """Two turns and a rest of the backward's workgroups."""
    print("case: layer norm, many rows", rows, C, dtype, flush=True)
    g = _gen(rows + C)
    x = (torch.randn(rows, C, generator=g) * 2 + torch.randn(C, generator=g)
         ).to(DT[dtype]).cuda()
    w = (1 + 0.2 * torch.randn(C, generator=g)).cuda()
    b = torch.randn(C, generator=g).cuda()
    dy = torch.randn(rows, C, generator=g).to(DT[dtype]).cuda()
    _check_norm(lm, x, w, b, dy)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_token_logprobs_gradients_of_many_rows(lm, dtype):
    """More tiles of a row than the gradient's grid has workgroups."""
    rows, V = (1 << 20) + 1003, 9
    print("case: token logprobs, many rows", rows, dtype, flush=True)
    g = _gen(17)
    x = _logits(g, rows, V, dtype=dtype).cuda()
    tok = torch.randint(-1, V, (rows,), generator=g)
    _check_score(lm, x, tok.cuda(), 0, 1.3)


def test_top_alternatives_far_from_zero(lm):
    """Distinct fp32 logits that share an offset: their order is in the low
    bits of their values."""
    for V in (300, 20011, 65536):
        x = 2 * torch.randn(3, V, generator=_gen(V))
        x[1] += 1000.0
        x[2] -= 4000.0
        tok = torch.zeros(3, dtype=torch.int64).cuda()
        for k in (1, 5, 64):
            print("case: far from zero", V, k, flush=True)
            _check_score(lm, x.cuda(), tok, k, grads=False)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [40, 700, 5003, 65536])
def test_certain_rows_are_certain(lm, V, dtype):
    """One token allowed, or one far above the rest: its log probability, the
    entropy, the loss of a teacher as sure and its gradients are exactly 0,
    and no log probability is above 0."""
    print("case: certain rows", V, dtype, flush=True)
    g = _gen(V)
    at = torch.randint(0, V, (64,), generator=g)
    size = (20 * torch.randn(64, 1, generator=g)).to(DT[dtype])
    x = torch.full((64, V), -INF).scatter_(1, at[:, None], size.float())
    x[32:][x[32:] == -INF] = -30000.0
    x = x.to(DT[dtype])
    for T in (1.0, 0.7, 1.3):
        leaf = x.cuda().requires_grad_()
        r = lm.token_logprobs(leaf, at.cuda(), top_k=3, temperature=T)
        assert not r.logprobs.any() and not r.entropy.any()
        assert torch.equal(r.top_ids[:, 0].cpu(), at)
        assert not r.top_logprobs[:, 0].any()
        d, = torch.autograd.grad((r.logprobs, r.entropy), leaf,
                                 [torch.ones(64).cuda()] * 2)
        assert not d.any()
        k = lm.distill_loss(leaf, at[:, None].cuda(), size.cuda(),
                            temperature=T)
        d, = torch.autograd.grad(k.loss, leaf)
        assert not k.loss.any() and not k.row_losses.any() and not d.any()
        y = (4 * torch.randn(64, V, generator=g)).to(DT[dtype])
        y[:, 0] += 16.0
        r = lm.token_logprobs(y.cuda(), torch.zeros_like(at).cuda(), top_k=3,
                              temperature=T)
        assert (r.logprobs <= 0).all() and (r.top_logprobs <= 0).all()
        assert (r.entropy >= 0).all()

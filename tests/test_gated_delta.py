"""The gated delta rule (gdr_*.hip) against the recurrence in float64, token by
token, and its gradients against that recurrence's and against differences.

Tolerances, relative to an output's largest magnitude.  With bf16 vectors a
computed operand is two bf16 planes and a product leaves out 2^-18 of each
operand, 2^-17 together; the longest way from an input to a result passes
eight products, whose roundings would add up to 8 * 2^-17 = 6e-5 if they all
agreed in sign: WIDE.  With fp32 vectors it is three planes and the sums' own
rounding, 2^-24 a term of up to 128 + 64 terms, sqrt of them as signs differ,
8 * 14 * 2^-24 = 7e-6, and exponentials of log decays 2^-23 a token of 64,
8e-6: NARROW is their sum.  bf16 results are rounded once more, 2^-8 of their
value.  dg is a running sum over a chunk of terms q.dq, beta k.left, k.right:
its tolerance goes by the largest of those times 8, the square root of 64.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
WIDE, NARROW = 6e-5, 1.5e-5
NAMES = ("q", "k", "v", "g", "beta")


@pytest.fixture(scope="module")
def lm(hip_lib):
    import rwkv7m_amd
    return rwkv7m_amd


def _gen(seed):
    return torch.Generator("cpu").manual_seed(seed)


def make(B, T, Hk, Hv, Dk, Dv, dtype, gtype="f32", seed=0, alike=0.7,
         decay=0.1):
    """CPU vectors and gates of the given types."""
    g = _gen(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g)

    q, k = normal(B, T, Hk, Dk), normal(B, T, Hk, Dk)
    k = k + alike * normal(B, 1, Hk, Dk)
    q, k = (x / x.norm(dim=-1, keepdim=True) for x in (q, k))
    v = normal(B, T, Hv, Dv)
    rate = decay * torch.exp(normal(Hv))
    gate = -rate * torch.nn.functional.softplus(normal(B, T, Hv))
    beta = torch.sigmoid(normal(B, T, Hv))
    return [q.to(DT[dtype]), k.to(DT[dtype]), v.to(DT[dtype]),
            gate.to(DT[gtype]), beta.to(DT[gtype])]


def rule64(q, k, v, g, beta, s0=None, scale=None):
    """The recurrence in float64 (differentiable by torch)."""
    per = v.shape[2] // q.shape[2]
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    q, k = (x.double().repeat_interleave(per, 2) for x in (q, k))
    v, a, beta = v.double(), g.double().exp(), beta.double()
    B, T, H, Dv = v.shape
    S = (torch.zeros(B, H, Dv, q.shape[-1], dtype=torch.float64)
         if s0 is None else s0.double())
    out = []
    for t in range(T):
        S = S * a[:, t, :, None, None]
        old = (S @ k[:, t, :, :, None])[..., 0]
        u = beta[:, t, :, None] * (v[:, t] - old)
        S = S + u[..., None] * k[:, t, :, None, :]
        out.append(scale * (S @ q[:, t, :, :, None])[..., 0])
    return (torch.stack(out, 1) if out else torch.zeros_like(v)), S


def grads64(inputs, s0, do, ds, scale=None):
    """([o, state], gradients of the five and of s0, sizes of dg's terms)."""
    leaves = [x.detach().double().requires_grad_() for x in inputs]
    per = inputs[2].shape[2] // inputs[0].shape[2]
    # q, k and their heads' copies apart, for the sizes of dg's terms
    start = None if s0 is None else s0.detach().double().requires_grad_()
    o, end = rule64(*leaves, start, scale)
    want = leaves + ([] if start is None else [start])
    grads = torch.autograd.grad(
        [o, end] if ds is not None else [o], want,
        [do.double(), ds.double()] if ds is not None else [do.double()],
        allow_unused=True)
    grads = [torch.zeros_like(x) if gr is None else gr
             for x, gr in zip(want, grads)]
    size = max(float((x * gr).detach().abs().sum(-1).max()) if x.numel() else 0.0
               for x, gr in zip(leaves[:3], grads[:3])) * per
    return [o.detach(), end.detach()], grads, size


def close(name, got, want, tol, size=None):
    got64, want = got.detach().double().cpu(), want.detach()
    assert got64.shape == want.shape, (name, got64.shape, want.shape)
    if not want.numel():
        return
    assert torch.isfinite(got64).all(), name
    size = float(want.abs().max()) if size is None else size
    bound = tol * size + (2.0 ** -8 * want.abs()
                          if got.dtype == torch.bfloat16 else 0.0)
    off = float(((got64 - want).abs() - bound).max())
    assert off <= 0, (name, off, size)


def tolerance(dtype):
    return WIDE if dtype == "bf16" else NARROW


def check(lm, inputs, s0, dtype, seed=0, with_end=True, scale=None,
          place=None):
    """Forward, state and every gradient of one call."""
    g = _gen(seed + 99)
    B, T, Hv, Dv = inputs[2].shape
    Dk = inputs[0].shape[-1]
    do = torch.randn(B, T, Hv, Dv, generator=g).to(inputs[2].dtype)
    ds = torch.randn(B, Hv, Dv, Dk, generator=g) if with_end else None
    (o, end), grads, size = grads64(inputs, s0, do, ds, scale)
    place = place or (lambda x: x.cuda())
    leaves = [place(x).detach().requires_grad_() for x in inputs]
    start = None if s0 is None else s0.cuda().requires_grad_()
    tol = tolerance(dtype)
    with torch.no_grad():
        o0, end0 = lm.gated_delta_rule(*leaves, start, scale)
    close("o", o0, o, tol)
    close("state", end0, end, tol)
    assert o0.dtype == inputs[2].dtype and end0.dtype == torch.float32
    o1, end1 = lm.gated_delta_rule(*leaves, start, scale)
    assert torch.equal(o0, o1) and torch.equal(end0, end1)
    outs, cots = [o1], [do.cuda()]
    if with_end:
        outs.append(end1)
        cots.append(ds.cuda())
    want = leaves + ([] if start is None else [start])
    got = torch.autograd.grad(outs, want, cots, retain_graph=True)
    for name, a, b in zip((*NAMES, "s0"), got, grads):
        close("d" + name, a, b, tol, 8 * size if name == "g" else None)
    again = torch.autograd.grad(outs, want, cots)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    for a, x in zip(got, want):
        assert a.dtype == x.dtype


# lengths around a chunk's 64 and a tile's 16 and 32 tokens
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 33, 48, 63, 64, 65, 100,
                               127, 128, 129, 200])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_lengths(lm, T, dtype):
    print("case: lengths", T, dtype, flush=True)
    x = make(2, T, 2, 2, 64, 64, dtype, seed=T)
    s0 = torch.randn(2, 2, 64, 64, generator=_gen(T + 1))
    check(lm, x, s0, dtype, T)


@pytest.mark.parametrize("Dk,Dv", [
    (8, 8), (16, 8), (8, 24), (24, 16), (40, 72), (56, 32), (64, 128),
    (72, 64), (88, 40), (96, 128), (104, 200), (120, 96), (128, 8),
    (128, 128), (128, 256), (64, 256)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_head_sizes(lm, Dk, Dv, dtype):
    print("case: head sizes", Dk, Dv, dtype, flush=True)
    x = make(1, 83, 1, 2, Dk, Dv, dtype, seed=Dk + Dv)
    s0 = torch.randn(1, 2, Dv, Dk, generator=_gen(Dv))
    check(lm, x, s0, dtype, Dk)


@pytest.mark.parametrize("B,Hk,Hv", [(1, 1, 1), (3, 1, 5), (2, 3, 9),
                                     (5, 2, 4), (1, 7, 7), (9, 1, 1)])
@pytest.mark.parametrize("dtype,gtype", [("bf16", "f32"), ("bf16", "bf16"),
                                         ("f32", "bf16")])
def test_heads_and_batches(lm, B, Hk, Hv, dtype, gtype):
    print("case: heads", B, Hk, Hv, dtype, gtype, flush=True)
    x = make(B, 70, Hk, Hv, 32, 48, dtype, gtype, seed=B * 10 + Hv)
    check(lm, x, None, dtype, B)
    check(lm, x, None, dtype, B, with_end=False)


# --- other layouts, gates and keys ------------------------------------------

def test_views_of_a_projection(lm):
    """Slices of one projection, time-major storage, gates of one tensor, and
    rows that have to be copied: as the same numbers in contiguous ones."""
    print("case: views", flush=True)
    B, T, Hk, Hv, Dk, Dv = 2, 90, 2, 4, 64, 32
    width = 2 * Hk * Dk + Hv * Dv
    flat = 0.1 * torch.randn(T, B, width + 24, generator=_gen(1))
    flat = flat.bfloat16().cuda()
    gates = torch.rand(T, B, 2 * Hv + 1, generator=_gen(2)).cuda()

    def views(off):
        x = flat[..., off:off + width].transpose(0, 1)
        q = x[..., :Hk * Dk].unflatten(-1, (Hk, Dk))
        k = x[..., Hk * Dk:2 * Hk * Dk].unflatten(-1, (Hk, Dk))
        v = x[..., 2 * Hk * Dk:].unflatten(-1, (Hv, Dv))
        g, beta = gates.transpose(0, 1)[..., 1:].chunk(2, -1)
        return q, k, v, -g, beta

    s0 = torch.randn(B * Hv * Dv * Dk + 1, generator=_gen(3)).cuda()
    for off in (0, 8, 3):  # (3: not 16-byte aligned)
        x = views(off)
        start = s0[off % 2:][:B * Hv * Dv * Dk].view(B, Hv, Dv, Dk)
        leaves = [t.detach().requires_grad_() for t in x]
        dense = [t.detach().contiguous().clone().requires_grad_() for t in x]
        a = lm.gated_delta_rule(*leaves, start)
        b = lm.gated_delta_rule(*dense, start.clone())
        do = torch.randn(T, B, Hv, Dv, generator=_gen(4)).bfloat16().cuda()
        ga = torch.autograd.grad(a[0], leaves, do.transpose(0, 1))
        gb = torch.autograd.grad(b[0], dense, do.transpose(0, 1).contiguous())
        for p, r in zip((*a, *ga), (*b, *gb)):
            assert torch.equal(p, r)
        # a broadcast cotangent, and a head of which all others are copies
        ga = torch.autograd.grad(lm.gated_delta_rule(*leaves)[0].sum(), leaves)
        gb = torch.autograd.grad(lm.gated_delta_rule(*dense)[0], dense,
                                 torch.ones_like(a[0]))
        assert all(torch.equal(p, r) for p, r in zip(ga, gb))
        wide = (leaves[0][:, :, :1].expand(-1, -1, Hk, -1),
                leaves[1][:, :, :1].expand(-1, -1, Hk, -1), *leaves[2:])
        with torch.no_grad():
            for p, r in zip(lm.gated_delta_rule(*wide),
                            lm.gated_delta_rule(*(t.contiguous()
                                                  for t in wide))):
                assert torch.equal(p, r)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gates_at_their_ends(lm, dtype):
    """Decays of 0 (log decay -inf and -1e30) clear the state, tokens with
    beta and g 0 leave it, and gradients stay finite."""
    print("case: gates", dtype, flush=True)
    x = make(2, 150, 1, 2, 64, 64, dtype, seed=3)
    g, beta = x[3], x[4]
    g[0, 70], g[1, 5], g[1, 128] = -float("inf"), -1e30, -float("inf")
    g[0, 100:], beta[0, 100:] = 0.0, 0.0
    g[1, 10:40], beta[1, 10:40] = 0.0, 1.0
    s0 = torch.randn(2, 2, 64, 64, generator=_gen(5))
    # the oracle's gradient of g at -inf is 0 times what is finite
    check(lm, x, s0, dtype, 1)
    cut = [t[:1, :100] for t in x]
    _, short = lm.gated_delta_rule(*(t.cuda() for t in cut), s0[:1].cuda())
    _, padded = lm.gated_delta_rule(*(t[:1].cuda() for t in x), s0[:1].cuda())
    close("padding", padded, short.double().cpu(), tolerance(dtype))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("decay", [0.0, 1e-3, 3.0])
def test_keys_alike_and_decays(lm, dtype, decay):
    """Keys that hardly differ (the inverse is then far from the identity),
    without a decay, with a slow one and a fast one."""
    print("case: keys alike", dtype, decay, flush=True)
    x = make(1, 200, 1, 2, 64, 64, dtype, seed=4, alike=6.0, decay=decay)
    check(lm, x, None, dtype, 2)


@pytest.mark.parametrize("scale", [1.0, 0.0, -2.5])
def test_scales(lm, scale):
    print("case: scale", scale, flush=True)
    check(lm, make(1, 66, 1, 1, 32, 32, "f32", seed=6), None, "f32", 3,
          scale=scale)


@pytest.mark.parametrize("B,T", [(0, 5), (2, 0), (0, 0)])
def test_nothing_to_do(lm, B, T):
    print("case: empty", B, T, flush=True)
    x = [t.cuda().requires_grad_() for t in make(B, T, 1, 2, 32, 16, "bf16")]
    s0 = torch.randn(B, 2, 16, 32, device="cuda", requires_grad=True)
    o, end = lm.gated_delta_rule(*x, s0)
    assert o.shape == (B, T, 2, 16) and torch.equal(end, s0)
    ds = torch.randn_like(end)
    *grads, d0 = torch.autograd.grad([o, end], [*x, s0],
                                     [torch.ones_like(o), ds])
    assert all(a.shape == b.shape for a, b in zip(grads, x))
    assert torch.equal(d0, ds)
    assert not lm.gated_delta_rule(*x)[1].any()
    state = torch.randn(B, 2, 16, 32, device="cuda")
    was = state.clone()
    with torch.no_grad():
        assert lm.gated_delta_step(*x, state).shape == (B, T, 2, 16)
    assert torch.equal(state, was)


def test_numbers_that_are_not_finite(lm):
    """They spoil what follows in their own heads and nothing before their
    chunk, in other heads or other sequences."""
    print("case: not finite", flush=True)
    x = [t.cuda() for t in make(2, 200, 2, 2, 64, 64, "bf16", seed=8)]
    o, end = lm.gated_delta_rule(*x)
    for which, bad in ((0, float("nan")), (1, float("inf")),
                       (2, -float("inf")), (3, float("nan")),
                       (4, float("nan"))):
        y = [t.clone() for t in x]
        y[which][0, 100, 1] = bad
        o2, end2 = lm.gated_delta_rule(*y)
        assert torch.equal(o2[1], o[1]) and torch.equal(end2[1], end[1])
        assert torch.equal(o2[0, :, 0], o[0, :, 0])
        assert torch.equal(end2[0, 0], end[0, 0])
        assert torch.equal(o2[0, :64, 1], o[0, :64, 1])
        if which == 0:
            assert torch.equal(end2, end)
            assert o2[0, 100, 1].isnan().all()
        else:
            assert o2[0, 100:, 1].isnan().any(-1).all()


def test_against_wkv7(lm):
    """As wkv7 with one decay a head, neg_kk = -k, kka = e^g beta k.  The
    other side rounds as much as this one: twice NARROW."""
    print("case: wkv7", flush=True)
    from rwkv7m_amd import wkv7_reference
    q, k, v, g, beta = make(2, 100, 2, 2, 64, 64, "f32", seed=9)
    s0 = torch.randn(2, 2, 64, 64, generator=_gen(1))
    o, end = lm.gated_delta_rule(*(t.cuda() for t in (q, k, v, g, beta)),
                                 s0.cuda(), 1.0)
    w = torch.log(-g)[..., None].expand_as(k)
    y, last = wkv7_reference(*(t.transpose(0, 1) for t in (
        q, w, beta[..., None] * k, v, -k,
        (g.exp() * beta)[..., None] * k)), s0)
    close("o", o, y.transpose(0, 1).double(), 2 * NARROW)
    close("state", end, last.double(), 2 * NARROW)


def test_pieces_of_a_sequence(lm):
    """One call, or several going on from each other's state."""
    print("case: pieces", flush=True)
    x = [t.cuda() for t in make(2, 300, 1, 3, 64, 40, "f32", seed=10)]
    o, end = lm.gated_delta_rule(*x)
    state, outs, at = None, [], 0
    for n in (64, 1, 100, 0, 135):
        part, state = lm.gated_delta_rule(*(t[:, at:at + n] for t in x), state)
        outs.append(part)
        at += n
    close("o", torch.cat(outs, 1), o.double().cpu(), 2 * NARROW)
    close("state", state, end.double().cpu(), 2 * NARROW)


def test_offsets_past_32_bits(lm):
    """Rows more than 2^32 bytes apart, and a pool of states as large: equal
    to the same rows close by, bit for bit."""
    print("case: offsets past 32 bits", flush=True)
    x = [t.cuda() for t in make(2, 70, 1, 1, 64, 64, "bf16", seed=11)]
    apart = 2 ** 31 + 64
    big = torch.zeros(apart + 70 * 192, dtype=torch.bfloat16, device="cuda")
    views = []
    for i in range(3):
        v = big.as_strided((2, 70, 1, 64), (apart, 192, 64, 1), 64 * i)
        v.copy_(x[i])
        views.append(v)
    for a, b in zip(lm.gated_delta_rule(*views, *x[3:]),
                    lm.gated_delta_rule(*x)):
        assert torch.equal(a, b)
    do = big.as_strided((2, 70, 1, 64), (apart, 192, 64, 1), 0)
    leaves = [t.detach().requires_grad_() for t in (*views, *x[3:])]
    near = [t.clone().requires_grad_() for t in x]
    for a, b in zip(
            torch.autograd.grad(lm.gated_delta_rule(*leaves)[0], leaves, do),
            torch.autograd.grad(lm.gated_delta_rule(*near)[0], near,
                                do.contiguous())):
        assert torch.equal(a, b)
    del big, views, leaves, do
    pool = torch.zeros(300000, 1, 64, 64, device="cuda")  # 4.6 GiB
    pool[-1].normal_()
    small = pool[-1:].clone()
    one = [t[:1, :2] for t in x]
    a = lm.gated_delta_step(*one, pool,
                            slots=torch.tensor([299999], device="cuda"))
    b = lm.gated_delta_step(*one, small)
    assert torch.equal(a, b) and torch.equal(pool[-1:], small)
    assert not pool[:-1].any()


# --- gradients ---------------------------------------------------------------

def test_gradients_against_differences(lm):
    """Central differences of a weighted sum of both outputs along random
    directions of unit norm, fp32.  With S the root of the sum's squared terms
    the rounding is at most 2 NARROW S over 2 h, 1.5e-3 S at h = 1e-2, and the
    truncation h^2 / 6 = 1.7e-5 of a third derivative of S's order: 3e-3 S."""
    print("case: differences", flush=True)
    x = [t.cuda() for t in make(1, 80, 1, 2, 32, 32, "f32", seed=12)]
    s0 = torch.randn(1, 2, 32, 32, generator=_gen(2)).cuda()
    wo = torch.randn(1, 80, 2, 32, generator=_gen(3)).cuda()
    ws = torch.randn(1, 2, 32, 32, generator=_gen(4)).cuda()

    def value(args):
        o, end = lm.gated_delta_rule(*args)
        return (o.double() * wo).sum() + (end.double() * ws).sum()

    leaves = [t.clone().requires_grad_() for t in (*x, s0)]
    o, end = lm.gated_delta_rule(*leaves)
    size = float((o * wo).detach().square().sum().sqrt()
                 + (end * ws).detach().square().sum().sqrt())
    grads = torch.autograd.grad([o, end], leaves, [wo, ws])
    h = 1e-2
    for i, gr in enumerate(grads):
        d = torch.randn(gr.shape, generator=_gen(20 + i)).cuda()
        d /= d.norm()
        up, down = ([t.detach() + (s * h * d if j == i else 0)
                     for j, t in enumerate(leaves)] for s in (1, -1))
        slope = float(value(up) - value(down)) / (2 * h)
        got = float((gr.double() * d).sum())
        assert abs(slope - got) <= 3e-3 * size, (i, slope, got, size)


def test_gradients_wanted_of_some(lm):
    """Any one input's gradient is that of all together; the state's, too."""
    print("case: some gradients", flush=True)
    x = [t.cuda() for t in make(1, 70, 1, 2, 32, 32, "bf16", seed=13)]
    x.append(torch.randn(1, 2, 32, 32, generator=_gen(1)).cuda())
    leaves = [t.clone().requires_grad_() for t in x]
    o, end = lm.gated_delta_rule(*leaves)
    do, ds = torch.randn_like(o), torch.randn_like(end)
    want = torch.autograd.grad([o, end], leaves, [do, ds])
    only = torch.autograd.grad(lm.gated_delta_rule(*leaves)[1], leaves, ds)
    zero = torch.autograd.grad([*lm.gated_delta_rule(*leaves)], leaves,
                               [torch.zeros_like(do), ds])
    assert all(torch.equal(a, b) for a, b in zip(only, zero))
    for i in range(6):
        mixed = [t.clone().requires_grad_(j == i) for j, t in enumerate(x)]
        o, end = lm.gated_delta_rule(*mixed)
        got, = torch.autograd.grad([o, end], [mixed[i]], [do, ds])
        assert torch.equal(got, want[i])


@pytest.mark.parametrize("B,T,Hk,Hv,Dk,Dv", [
    (1, 84, 2, 6, 64, 64), (5, 203, 3, 3, 128, 256), (3, 300, 1, 3, 64, 128)])
def test_fp32_results_of_bf16_vectors(lm, B, T, Hk, Hv, Dk, Dv):
    """By their 2-norms.  Two planes leave out 2^-18 of an operand's place at
    most, 2^-18 / sqrt(3) in the mean, and the product of the second planes as
    much: with eight products on the longest way 4 2^-18 / sqrt(3) sqrt(2) =
    1.2e-5 if all had that mean; most places are further from a rounding's
    border and the ways mostly shorter: 1e-5.  dg is <D, S (I - beta k k^T)> of
    a token, factor by factor a product of two results off by 1.2e-5, each
    place by itself: sqrt(2) 1.2e-5 = 1.7e-5 of the sum's size."""
    print("case: fp32 results", B, T, Hk, Hv, Dk, Dv, flush=True)
    x = make(B, T, Hk, Hv, Dk, Dv, "bf16", seed=T)
    s0 = torch.randn(B, Hv, Dv, Dk, generator=_gen(1))
    do = torch.randn(B, T, Hv, Dv, generator=_gen(2)).bfloat16()
    ds = torch.randn(B, Hv, Dv, Dk, generator=_gen(3))
    (_, end), grads, _ = grads64(x, s0, do, ds)
    leaves = [t.cuda().requires_grad_() for t in (*x, s0)]
    o, got = lm.gated_delta_rule(*leaves)
    d = torch.autograd.grad([o, got], leaves, [do.cuda(), ds.cuda()])
    for name, a, b in (("state", got, end), ("dg", d[3], grads[3]),
                       ("dbeta", d[4], grads[4]), ("ds0", d[5], grads[5])):
        off = float((a.detach().double().cpu() - b).norm() / b.norm())
        assert off <= (1.7e-5 if name == "dg" else 1e-5), (name, off)


def test_derivatives_that_are_refused(lm):
    print("case: derivatives refused", flush=True)
    x = [t.cuda().requires_grad_() for t in make(1, 5, 1, 1, 16, 16, "f32")]
    out = lm.gated_delta_rule(*x)[0].square().sum()
    d, = torch.autograd.grad(out, x[0], create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not "
                                           "require grad"):
        d.sum().backward()
    state = torch.zeros(1, 1, 16, 16, device="cuda")
    with pytest.raises(RuntimeError, match="no gradient"):
        lm.gated_delta_step(*x, state)
    import torch.autograd.forward_ad as fwd
    with torch.no_grad(), fwd.dual_level():
        y = [t.detach() for t in x]
        y[1] = fwd.make_dual(y[1], torch.ones_like(y[1]))
        for call in (lambda: lm.gated_delta_rule(*y),
                     lambda: lm.gated_delta_step(*y, state)):
            with pytest.raises(TypeError, match="forward-mode"):
                call()
    # what a backward saved and a step then changes is noticed
    state = torch.randn(1, 1, 16, 16, device="cuda")
    w = torch.ones_like(state, requires_grad=True)
    kept = (state * w).sum()
    with torch.no_grad():
        lm.gated_delta_step(*x, state, update_state=False)
    kept.backward(retain_graph=True)
    with torch.no_grad():
        lm.gated_delta_step(*x, state)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        kept.backward()

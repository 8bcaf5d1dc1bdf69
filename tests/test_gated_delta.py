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
    size = max(float((x * gr).abs().sum(-1).max()) if x.numel() else 0.0
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

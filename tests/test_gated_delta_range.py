"""The gated delta rule over the whole range that it is documented for: what its
fp32 results are off by, rates (beta) up to 2, keys that hardly differ, and
calls large enough for every division of a sequence's work.

Tolerances, of 2-norms.  A product adds up at most 128 + 64 terms in 24 fp32
additions of a matrix instruction's sums (4 tiles of 32 places, six products of
planes each), each off by 2^-24 / sqrt(3) in the mean: 1.7e-7.  The longest way
from an input to a result passes eight products, sqrt(8) 1.7e-7 = 4.8e-7, and
exponentials of up to 8 in base 2 (smaller weights do not count), 2^-24 8 ln 2 /
sqrt(3) = 2e-7; a row of the inverse, whose places are as large as beta, doubles
what comes to it: 1.4e-6, FP32 = 1.5e-6.  dg is the running sum of three such
terms that cancel: sqrt(3) FP32.  Where beta is up to 2 or keys hardly differ, the
64 terms of a row of the inverse times what it acts on are each as large as the
result and differ in sign: sqrt(64) as much.
"""

from __future__ import annotations

import pytest
import torch

from test_gated_delta import _gen, close, grads64, make

pytestmark = pytest.mark.gpu

FP32 = 1.5e-6


@pytest.fixture(scope="module")
def lm(hip_lib):
    import rwkv7m_amd
    return rwkv7m_amd


def results(lm, x, s0, seed):
    """{name: (got, wanted)} of the fp32 results, and the bf16 ones compared."""
    g = _gen(seed)
    B, T, Hv, Dv = x[2].shape
    do = torch.randn(B, T, Hv, Dv, generator=g).to(x[2].dtype)
    ds = torch.randn(s0.shape, generator=g)
    (o, end), grads, _ = grads64(x, s0, do, ds)
    leaves = [t.cuda().requires_grad_() for t in (*x, s0)]
    out, got = lm.gated_delta_rule(*leaves)
    d = torch.autograd.grad([out, got], leaves, [do.cuda(), ds.cuda()])
    return dict(o=(out, o), state=(got, end), dq=(d[0], grads[0]),
                dk=(d[1], grads[1]), dv=(d[2], grads[2]),
                dg=(d[3], grads[3]), dbeta=(d[4], grads[4]),
                ds0=(d[5], grads[5]))


def check_norms(found, factor):
    for name, (got, want) in found.items():
        got = got.detach()
        if got.dtype == torch.bfloat16:
            close(name, got, want, 16 * factor * FP32)
            continue
        off = float((got.double().cpu() - want).norm() / want.norm())
        tol = factor * FP32 * (3 ** 0.5 if name == "dg" else 1.0)
        assert off <= tol, (name, off, tol)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,T,Hk,Hv,Dk,Dv", [
    (1, 84, 2, 6, 64, 64), (2, 203, 2, 2, 128, 128), (2, 300, 1, 3, 40, 72)])
def test_fp32_results_as_of_fp32_products(lm, B, T, Hk, Hv, Dk, Dv, dtype):
    print("case: fp32 results", B, T, Hk, Hv, Dk, Dv, dtype, flush=True)
    x = make(B, T, Hk, Hv, Dk, Dv, dtype, seed=T)
    s0 = torch.randn(B, Hv, Dv, Dk, generator=_gen(1))
    check_norms(results(lm, x, s0, 2), 1.0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("alike,decay", [(0.7, 0.0), (0.7, 0.1), (6.0, 0.0),
                                         (6.0, 0.1)])
@pytest.mark.parametrize("D", [64, 128])
def test_rates_up_to_two(lm, dtype, alike, decay, D):
    """beta from 1 to 2, keys of length 1: reflections, next to no decay."""
    print("case: rates", dtype, alike, decay, D, flush=True)
    x = make(2, 200, 2, 2, D, 64, dtype, seed=5, alike=alike, decay=decay)
    x[4] = 1.0 + torch.rand(x[4].shape, generator=_gen(6))
    if dtype == "bf16":  # keys of at most length 1 after their rounding
        x[1] = (x[1].float() * (1 - 2.0 ** -8)).bfloat16()
    s0 = torch.randn(2, 2, 64, D, generator=_gen(7))
    check_norms(results(lm, x, s0, 8), 8.0)


# --- layouts ------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_dense_tensors_that_start_anywhere(lm, dtype):
    """Contiguous vectors, cotangents and gates an element past a 16-byte
    border: as the same numbers at one."""
    print("case: odd starts", dtype, flush=True)

    def odd(t):
        out = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:]
        out = out.view(t.shape).copy_(t)
        assert out.is_contiguous() and out.data_ptr() % 16
        return out

    x = make(2, 70, 1, 2, 32, 40, dtype, seed=21)
    s0 = torch.randn(2, 2, 40, 32, generator=_gen(1))
    do = torch.randn(2, 70, 2, 40, generator=_gen(2)).to(x[2].dtype)
    ds = torch.randn(2, 2, 40, 32, generator=_gen(3))
    found = []
    for place in (lambda t: t.cuda(), odd):
        leaves = [place(t).requires_grad_() for t in (*x, s0)]
        out = lm.gated_delta_rule(*leaves)
        found.append([*out, *torch.autograd.grad(out, leaves,
                                                 [place(do), place(ds)])])
        with torch.no_grad():
            found[-1] += lm.gated_delta_rule(*leaves)
            state = s0.cuda()
            found[-1] += [lm.gated_delta_step(*(t[:, :3] for t in leaves[:5]),
                                              state), state]
            one = [place(t[:, 5:6].contiguous()) for t in x]
            state = s0.cuda()
            found[-1] += [lm.gated_delta_step(*one, state), state]
    for a, b in zip(*found):
        assert torch.equal(a, b)


# --- division of work ---------------------------------------------------------

# heads and Dv choose how many waves of a workgroup own rows of the state (on
# 256 CUs, as the name says); in some cases the last workgroup of a head has
# waves past its rows
@pytest.mark.parametrize("Dk", [64, 72, 128])
@pytest.mark.parametrize("B,Hk,Hv,T,Dv", [
    pytest.param(16, 3, 6, 70, 64, id="two"),
    pytest.param(16, 5, 5, 70, 40, id="two-part-of-a-tile"),
    pytest.param(16, 2, 4, 130, 96, id="two-three-workgroups"),
    pytest.param(5, 2, 6, 70, 200, id="two-of-224-rows"),
    pytest.param(24, 4, 4, 70, 72, id="four-two-past-the-rows"),
    pytest.param(24, 2, 4, 70, 200, id="four-of-224-rows"),
    pytest.param(75, 4, 4, 70, 32, id="four-two-idle"),
    pytest.param(48, 1, 2, 129, 128, id="four"),
    pytest.param(33, 8, 8, 66, 256, id="four-256-rows")])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_many_heads(lm, dtype, B, Hk, Hv, T, Dv, Dk):
    """Sequences of a large batch against the recurrence, and bit for bit
    against the same ones in calls of their own."""
    print("case: many heads", dtype, B, Hk, Hv, T, Dk, Dv, flush=True)
    x = make(B, T, Hk, Hv, Dk, Dv, dtype, seed=Dk + Dv)
    s0 = torch.randn(B, Hv, Dv, Dk, generator=_gen(1))
    do = torch.randn(B, T, Hv, Dv, generator=_gen(2)).to(x[2].dtype)
    ds = torch.randn(B, Hv, Dv, Dk, generator=_gen(3))

    def call(rows):
        leaves = [t[rows].cuda().requires_grad_() for t in (*x, s0)]
        with torch.no_grad():
            plain = lm.gated_delta_rule(*leaves)
        out = lm.gated_delta_rule(*leaves)
        assert all(torch.equal(a, b) for a, b in zip(plain, out))
        return [*out, *torch.autograd.grad(
            out, leaves, [do[rows].cuda(), ds[rows].cuda()])]

    names = ("o", "state", "dq", "dk", "dv", "dg", "dbeta", "ds0")
    whole = call(slice(None))
    for b in (0, B // 2, B - 1):
        rows = slice(b, b + 1)
        alone = call(rows)
        for name, a, c in zip(names, whole, alone):
            assert torch.equal(a[rows], c), (name, b)
        outs, grads, _ = grads64([t[rows] for t in x], s0[rows], do[rows],
                                 ds[rows])
        check_norms({n: (a[rows], w) for n, a, w in
                     zip(names, whole, [*outs, *grads])}, 1.0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_broadcast_gates_and_cotangents(lm, dtype):
    """One gate for all heads or tokens, one key for all, and the cotangents of
    sums (all of one number): as the same ones written out."""
    print("case: broadcast", dtype, flush=True)
    q, k, v, g, beta = (t.cuda() for t in make(2, 100, 2, 4, 64, 32, dtype,
                                               seed=31))
    s0 = torch.randn(1, 4, 32, 64, generator=_gen(1)).cuda()
    s0 = s0.expand(2, -1, -1, -1)
    x = (q[:1].expand(2, -1, -1, -1), k[:, :1].expand(-1, 100, -1, -1),
         v[:, :, :1].expand(-1, -1, 4, -1), g[..., :1].expand(-1, -1, 4),
         beta[:, :1].expand(-1, 100, -1), s0)
    found = []
    for place in (lambda t: t.detach(), lambda t: t.detach().contiguous()):
        leaves = [place(t).requires_grad_() for t in x]
        o, end = lm.gated_delta_rule(*leaves)
        ones = [place(t.new_ones(()).expand(t.shape)) for t in (o, end)]
        found.append([o, end, *torch.autograd.grad((o, end), leaves, ones)])
        state = s0.contiguous()
        with torch.no_grad():
            found[-1] += [lm.gated_delta_step(*(t[:, :4] for t in leaves[:5]),
                                              state), state]
    for a, b in zip(*found):
        assert torch.equal(a, b)

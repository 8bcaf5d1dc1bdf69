"""Verification of drafted tokens: derivatives that are refused (without a GPU),
and on the GPU what is drawn where nothing is left, drafts outside the
vocabulary next to greedy ones and rows without a distribution, and calls of
more workgroups than one row of a grid holds."""

from __future__ import annotations

import pytest
import torch

from rwkv7m_amd import verify_drafts


def test_derivatives_are_refused():
    """Neither tangents nor gradients are dropped; no valid request is made
    (CPU tensors are refused last)."""
    x, tok = torch.randn(2, 4, 50), torch.zeros(2, 3, dtype=torch.int64)
    u, s = torch.rand(2, 3), torch.rand(2)
    y = x[:, :3].clone()
    import torch.autograd.forward_ad as fwd
    args = dict(logits=x, draft_tokens=tok, draft_logits=y, accept_uniforms=u,
                sample_uniforms=s)
    for name in ("logits", "draft_logits", "accept_uniforms",
                 "sample_uniforms"):
        with torch.no_grad(), fwd.dual_level():
            dual = fwd.make_dual(args[name], torch.ones_like(args[name]))
            with pytest.raises(TypeError, match="verify_drafts.*forward-mode"):
                verify_drafts(**{**args, name: dual})
        leaf = args[name].clone().requires_grad_()
        with pytest.raises(RuntimeError, match="has no gradient"):
            verify_drafts(**{**args, name: leaf})
        with pytest.raises(RuntimeError, match="has no gradient"):
            verify_drafts(**{**args, name: leaf * 1})
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU tensors"):
            verify_drafts(**{**args, name: leaf})
        with pytest.raises(RuntimeError, match="GPU tensors"):
            verify_drafts(**{**args, name: leaf.detach()})


@pytest.fixture(scope="module")
def lm(hip_lib):
    import rwkv7m_amd
    return rwkv7m_amd


def _call(lm, x, tok, y=None, u=None, s=None, temp=1.0, n=None):
    B, K = tok.shape
    u = torch.zeros(B, K) if u is None else u
    s = torch.zeros(B) if s is None else s
    got = lm.verify_drafts(x.cuda(), tok.cuda(),
                           None if y is None else y.cuda(), u.cuda(),
                           s.cuda(), None if n is None else n.cuda(), temp)
    return [t.cpu() for t in got]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_greedy_drafts_outside_the_vocabulary(lm, dtype):
    print("case: greedy, outside", dtype, flush=True)
    x = torch.randn(4, 3, 500, generator=torch.Generator().manual_seed(4))
    x = x.to(dtype)
    best = x.double().argmax(-1)
    tok = best[:, :2].clone()
    tok[0, 0], tok[1, 0], tok[2, 1], tok[3, 0] = -1, 500, 2 ** 40, -2 ** 62
    took, count, chance = _call(lm, x, tok, temp=0.0)
    assert count.tolist() == [0, 0, 1, 0]
    assert took.tolist() == [
        [int(best[0, 0]), -1, -1], [int(best[1, 0]), -1, -1],
        [int(best[2, 0]), int(best[2, 1]), -1], [int(best[3, 0]), -1, -1]]
    assert chance.tolist() == [[0.0, 1.0], [0.0, 1.0], [1.0, 0.0], [0.0, 1.0]]


@pytest.mark.gpu
@pytest.mark.parametrize("temp", [0.0, 1.0])
@pytest.mark.parametrize("what", ["nan", "inf", "empty"])
def test_drafts_outside_the_vocabulary_of_rows_without_a_distribution(
        lm, temp, what):
    """The chance is NaN there, as of any other draft, and the token is -1."""
    print("case: outside, no distribution", temp, what, flush=True)
    g = torch.Generator().manual_seed(5)
    x, y = torch.randn(3, 2, 300, generator=g), torch.randn(3, 1, 300,
                                                            generator=g)
    tok = torch.tensor([[-1], [300], [-1]])

    def spoiled(t):
        t = t.clone()
        t[:2, 0] = -float("inf") if what == "empty" else t[:2, 0]
        if what != "empty":
            t[:2, 0, 7] = float(what)
        return t

    for a, q in ((spoiled(x), None), (spoiled(x), y), (x, spoiled(y))):
        if temp == 0.0 and a is x:
            continue  # (the draft's logits are not looked at)
        took, count, chance = _call(lm, a, tok, q, temp=temp)
        assert count.tolist() == [0, 0, 0]
        assert took[:2].tolist() == [[-1, -1]] * 2 and 0 <= took[2, 0] < 300
        assert chance[:2].isnan().all() and float(chance[2, 0]) == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("B,K", [(25000, 1), (70000, 0), (66000, 2)])
@pytest.mark.parametrize("kind", ["drawn", "certain", "greedy"])
def test_more_workgroups_than_a_grid_row(lm, B, K, kind):
    """More than 2^16 workgroups in either launch: sequences from the start, the
    middle and the end as in small calls."""
    print("case: grid rows", B, K, kind, flush=True)
    V = 33
    g = torch.Generator("cuda").manual_seed(B)
    x = 2 * torch.randn(B, K + 1, V, generator=g, device="cuda")
    y = x[:, :K] + torch.randn(B, K, V, generator=g, device="cuda")
    tok = torch.randint(0, V, (B, K), generator=g, device="cuda")
    u = torch.rand(B, K, generator=g, device="cuda")
    s = torch.rand(B, generator=g, device="cuda")
    n = torch.randint(0, K + 1, (B,), generator=g, device="cuda")
    temp = 0.0 if kind == "greedy" else 1.0
    q = y if kind == "drawn" else None
    got = lm.verify_drafts(x, tok, q, u, s, n, temp)
    for a in (0, B // 2, 65530, 21840, B - 40):
        if a > B - 40:
            continue
        r = slice(a, a + 40)
        part = lm.verify_drafts(x[r], tok[r], None if q is None else q[r],
                                u[r], s[r], n[r], temp)
        for p, w in zip(got, part):
            assert torch.equal(p[r], w)
    # every sequence has its token, and no draft past its length is taken
    assert bool((got.accepted <= n).all())
    last = got.tokens.gather(1, got.accepted[:, None])
    assert bool((last >= 0).all()) and bool((last < V).all())
    if temp == 0.0:
        want = x.gather(1, got.accepted[:, None, None].expand(-1, 1, V))
        assert torch.equal(last[:, 0], want[:, 0].argmax(-1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [7, 9000])
def test_what_is_drawn_where_nothing_is_left(lm, dtype, V):
    """A draft that is not taken though p = q: the token comes from p."""
    print("case: nothing left", dtype, V, flush=True)
    g = torch.Generator().manual_seed(V)
    x = torch.randn(1, 2, V, generator=g).to(dtype).expand(9, 2, V)
    tok = torch.full((9, 1), V)
    s = torch.linspace(0.0, 0.999, 9)
    took, count, chance = _call(lm, x, tok, x[:, :1], s=s)
    assert not count.any() and not chance.any()
    cum = torch.softmax(x[0, 0].double(), -1).cumsum(-1)
    at = s.double() * cum[-1]
    assert float((cum[None] - at[:, None]).abs().min(-1).values[1:].min()) \
        > 1e-9
    assert took[:, 0].tolist() == (cum[None] <= at[:, None]).sum(-1).tolist()
    assert (took[:, 1] == -1).all()
    # without a draft's logits p itself is drawn from: nothing is set aside
    other, *_ = _call(lm, x, tok, s=s)
    assert torch.equal(took, other)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ends_of_the_temperatures(lm, dtype):
    """At 1e-30 as the greedy form, whatever the random numbers and however far
    the logits, at 1e30 as a flat row."""
    print("case: temperatures", dtype, flush=True)
    g = torch.Generator().manual_seed(8)
    V = 9001
    x = (3e37 * torch.randn(6, 3, V, generator=g)).to(dtype)
    x[:, :, 8999] = 3e38  # (one likeliest token each)
    x[3:, 1, 8999], x[3:, 1, 17] = -float("inf"), 3.1e38
    tok = torch.full((6, 2), 8999)
    u, s = torch.rand(6, 2, generator=g), torch.rand(6, generator=g)
    cold = _call(lm, x, tok, None, u, s, 1e-30)
    greedy = _call(lm, x, tok, temp=0.0)
    assert all(torch.equal(a, b) for a, b in zip(cold, greedy))
    assert cold[1].tolist() == [2, 2, 2, 1, 1, 1]
    flat = torch.randn(6, 1, V, generator=g).to(dtype)
    took, *_ = _call(lm, flat, torch.zeros(6, 0).long(), None,
                     torch.zeros(6, 0), s, 1e30)
    # (a flat row's running sum is the id, but for rounding)
    assert bool(((took[:, 0] - (s.double() * V).floor()).abs() <= 1).all())


@pytest.mark.gpu
def test_a_vocabulary_of_a_million(lm):
    print("case: a million", flush=True)
    g = torch.Generator().manual_seed(9)
    V = 1000003
    x = torch.randn(2, 2, V, generator=g)
    tok = torch.tensor([[V - 1], [5]])
    s = torch.tensor([0.25, 0.999])
    took, count, chance = _call(lm, x, tok, None, torch.full((2, 1), 0.5), s)
    p = torch.softmax(x.double(), -1)
    assert not count.any()
    off = chance[:, 0].double() - p[[0, 1], 0, tok[:, 0]]
    assert float(off.abs().max()) <= 1e-7 * float(chance.max())
    p[[0, 1], 0, tok[:, 0]] = 0.0
    cum = p[:, 0].cumsum(-1)
    at = s.double()[:, None] * cum[:, -1:]
    assert float((cum - at).abs().min()) > 1e-9
    assert took[:, 0].tolist() == (cum <= at).sum(-1).tolist()

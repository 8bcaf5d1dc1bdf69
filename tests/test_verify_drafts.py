"""Verification of drafted tokens (lm_verify.hip) against the rule in float64
on the CPU.

Whole numbers are equal: every case's random numbers keep 1e-9 away from the
borders that decide (checked in the oracle; exponentials and sums are off by
some 1e-12), or lie on them exactly where the rule says what follows.  Chances
are a quotient rounded to fp32, 2^-24 of them, next to 1e-11 of sums: 1e-7.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
INF = float("inf")


@pytest.fixture(scope="module")
def lm(hip_lib):
    import rwkv7m_amd
    return rwkv7m_amd


def _gen(seed):
    return torch.Generator("cpu").manual_seed(seed)


def make(B, K, V, dtype, seed, certain=False, spread=2.0):
    g = _gen(seed)
    x = spread * torch.randn(B, K + 1, V, generator=g)
    at = torch.randint(0, V, (B, K + 1, 3), generator=g)
    x.scatter_(-1, at, 6.0 + torch.randn(B, K + 1, 3, generator=g))
    y = x[:, :K] + 0.7 * torch.randn(B, K, V, generator=g)
    x, y = x.to(DT[dtype]), y.to(DT[dtype])
    p = torch.softmax(y.double(), -1)
    tok = torch.multinomial(p.reshape(-1, V).clamp(min=1e-300), 1,
                            generator=g).view(B, K) if K else \
        torch.zeros(B, 0, dtype=torch.int64)
    u = torch.rand(B, K, generator=g)
    s = torch.rand(B, generator=g)
    return x, tok, None if certain else y, u, s


def rule(x, tok, y, u, s, n=None, temp=1.0):
    """(tokens, accepted, chances) by the definition, one sequence at a time;
    asserts that no random number lies within 1e-9 of what it decides."""
    B, K1, V = x.shape
    K = K1 - 1
    out = torch.full((B, K1), -1, dtype=torch.int64)
    took, prob = torch.zeros(B, dtype=torch.int64), torch.zeros(B, K).double()
    for b in range(B):
        count = K if n is None else min(max(int(n[b]), 0), K)
        if temp == 0.0:
            best = [int(x[b, i].double().argmax()) for i in range(K1)]
            m = 0
            while m < count and int(tok[b, m]) == best[m]:
                m += 1
            for i in range(count):
                prob[b, i] = float(int(tok[b, i]) == best[i])
            out[b, :m], out[b, m], took[b] = tok[b, :m], best[m], m
            continue
        p = torch.softmax(x[b].double() / temp, -1)
        q = torch.zeros(K, V).double()
        if y is not None:
            q = torch.softmax(y[b].double() / temp, -1)
        m, going = 0, True
        for i in range(count):
            t = int(tok[b, i])
            inside = 0 <= t < V
            if y is None and inside:
                q[i, t] = 1.0
            px = float(p[i, t]) if inside else 0.0
            qx = float(q[i, t]) if inside else 1.0
            prob[b, i] = min(1.0, px / qx) if qx else float(px > 0)
            left = float(u[b, i].double()) * qx
            if going:
                assert abs(left - px) > 1e-9 * px or px == 0.0
                if left < px:
                    m += 1
                else:
                    going = False
        r = p[m] - q[m] if m < count else p[m]
        r = r.clamp(min=0.0)
        if not float(r.sum()) > 0:
            r = p[m]
        cum = r.cumsum(-1)
        at = float(s[b].double()) * float(cum[-1])
        gap = float((cum - at).abs().min())
        assert gap > 1e-9 * float(cum[-1]) or at == 0.0
        out[b, :m] = tok[b, :m]
        out[b, m] = int(((cum <= at) | (r == 0)).long().cumprod(-1).sum()) \
            if at == 0.0 else int((cum <= at).sum())
        took[b] = m
    return out, took, prob


def check(lm, x, tok, y, u, s, n=None, temp=1.0, place=lambda t: t.cuda()):
    want = rule(x, tok, y, u, s, n, temp)
    args = (place(x), tok.cuda(), None if y is None else place(y), u.cuda(),
            s.cuda(), None if n is None else n.cuda(), temp)
    got = lm.verify_drafts(*args)
    assert got.tokens.dtype == got.accepted.dtype == torch.int64
    assert torch.equal(got.accepted.cpu(), want[1])
    assert torch.equal(got.tokens.cpu(), want[0])
    off = (got.chances.double().cpu() - want[2]).abs()
    assert not off.numel() or float(off.max()) <= 1e-7
    again = lm.verify_drafts(*args)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    return got


@pytest.mark.parametrize("V", [1, 2, 7, 255, 256, 257, 511, 513, 4095, 8191,
                               8192, 8193, 16391, 65529, 65536, 131075])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_vocabularies(lm, V, dtype):
    print("case: vocabulary", V, dtype, flush=True)
    check(lm, *make(5, 3, V, dtype, V))


@pytest.mark.parametrize("B,K", [(1, 0), (1, 1), (7, 2), (2, 15), (2, 16),
                                 (1, 33), (1, 64), (70, 4)])
@pytest.mark.parametrize("certain", [False, True])
def test_drafts_and_batches(lm, B, K, certain):
    print("case: drafts", B, K, certain, flush=True)
    x, tok, y, u, s = make(B, K, 1001, "bf16", 10 * B + K, certain)
    check(lm, x, tok, y, u, s)
    # all taken: the token behind is drawn from the last row
    got = check(lm, x, tok, y, u * 0, s, temp=1.0)
    assert int(got.accepted.min()) == K


@pytest.mark.parametrize("temp", [0.0, 0.3, 1.0, 3.0])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_ragged_and_temperatures(lm, temp, dtype):
    print("case: ragged", temp, dtype, flush=True)
    x, tok, y, u, s = make(24, 6, 9000, dtype, 5)
    tok[::2, :3] = x[::2, :3].double().argmax(-1)
    n = torch.randint(-1, 9, (24,), generator=_gen(6))
    check(lm, x, tok, y, u, s, n, temp)
    check(lm, x, tok.int(), y, u, s, n.int(), temp)
    check(lm, x, tok, None, u, s, n, temp)


# --- rows at their ends --------------------------------------------------------

def _one(lm, x, tok, y=None, u=None, s=None, temp=1.0):
    B, K = tok.shape
    u = torch.zeros(B, K) if u is None else u
    s = torch.zeros(B) if s is None else s
    got = lm.verify_drafts(x.cuda(), tok.cuda(),
                           None if y is None else y.cuda(), u.cuda(),
                           s.cuda(), None, temp)
    return [t.cpu() for t in got]


@pytest.mark.parametrize("V", [300, 9000])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("masked", [-INF, None])
def test_masked_tokens(lm, V, dtype, masked):
    """Nothing masked, by -inf or the type's lowest value, is taken or drawn,
    not by random numbers of 0 or next to 1 either."""
    print("case: masks", V, dtype, masked, flush=True)
    low = torch.finfo(DT[dtype]).min if masked is None else masked
    x = torch.full((4, 3, V), low, dtype=DT[dtype])
    y = x[:, :2].clone()
    allowed = [3, V // 2, V - 2]
    x[..., allowed] = torch.tensor([0.5, 1.0, -1.0], dtype=DT[dtype])
    y[..., allowed] = torch.tensor([1.0, -2.0, -1.0], dtype=DT[dtype])
    tok = torch.tensor([[allowed[0], 0], [0, 1], [V - 1, 3], [3, V // 2]])
    top = torch.tensor(1.0 - 2.0 ** -24)
    for s in (torch.zeros(4), top.expand(4).clone()):
        for q in (None, y):
            took, count, chance = (t for t in _one(lm, x, tok, q, None, s))
            assert count.tolist() == [1, 0, 0, 2]
            drawn = took.gather(1, count[:, None])[:, 0]
            assert set(drawn.tolist()) <= set(allowed)
            assert (took[took >= 0][:, None] ==
                    torch.tensor(allowed)).any(-1).all()
            if q is None:  # row 0 draws without token 0, which has nothing
                last = allowed[0] if float(s[0]) == 0.0 else allowed[2]
                assert drawn.tolist()[:3] == [last] * 3
            assert chance[1].tolist() == [0.0, 0.0] or q is not None
    # certain drafts refused: the drawn token is another one
    two = torch.full((1, 2, V), low, dtype=DT[dtype])
    two[..., [5, 7]] = 0.0
    for s in (0.0, 0.5, float(top)):
        took, count, _ = _one(lm, two, torch.tensor([[5]]), None,
                              torch.full((1, 1), 0.75), torch.tensor([s]))
        assert int(count) == 0 and took.tolist() == [[7, -1]]
    # one token left in the vocabulary
    two[..., 7] = low
    took, count, chance = _one(lm, two, torch.tensor([[5]]), two[:, :1],
                               torch.full((1, 1), 0.75), torch.tensor([0.9]))
    assert took.tolist() == [[5, 5]] and float(chance) == 1.0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("temp", [0.0, 0.7])
@pytest.mark.parametrize("what", ["nan", "inf", "empty"])
def test_rows_without_a_distribution(lm, dtype, temp, what):
    print("case: no distribution", dtype, temp, what, flush=True)
    V = 8200
    x, tok, y, u, s = make(3, 2, V, dtype, 3)
    tok[:] = x[:, :2].double().argmax(-1)
    u *= 0

    def spoil(row):
        if what == "empty":
            row[:] = -INF
        else:
            row[8195] = float(what)

    for spoiled in range(3):
        bad = x.clone()
        spoil(bad[1, spoiled])
        for q in (None, y):
            took, count, chance = _one(lm, bad, tok, q, u, s, temp)
            good = _one(lm, x, tok, q, u, s, temp)
            assert int(count[1]) == spoiled
            assert took[1].tolist() == tok[1, :spoiled].tolist() + \
                [-1] * (3 - spoiled)
            if spoiled < 2:
                assert chance[1, spoiled].isnan()
            for a, b in zip((took, count, chance), good):
                assert torch.equal(a[[0, 2]], b[[0, 2]])
    if temp:
        bad = y.clone()
        spoil(bad[1, 0])
        took, count, chance = _one(lm, x, tok, bad, u, s, temp)
        assert int(count[1]) == 0 and took[1].tolist() == [-1] * 3
        assert chance[1, 0].isnan()


def test_drafts_outside_the_vocabulary(lm):
    print("case: outside", flush=True)
    x, tok, y, u, s = make(4, 2, 500, "f32", 4)
    tok[0, 0], tok[1, 0], tok[2, 1], tok[3, 0] = -1, 500, 2 ** 40, -2 ** 62
    u *= 0
    for q in (None, y):
        took, count, chance = _one(lm, x, tok, q, u, s)
        assert count.tolist() == [0, 0, 1, 0]
        assert chance[[0, 1, 2, 3], [0, 0, 1, 0]].tolist() == [0.0] * 4
        assert bool((took.gather(1, count[:, None]) >= 0).all())
    took, count, _ = _one(lm, x, tok, temp=0.0)
    assert count.tolist() == [0, 0, 0, 0] or int(tok[2, 0]) == int(took[2, 0])


def test_equal_rows_and_ties(lm):
    """p = q: nothing is left, every draft is taken below 1; equal logits:
    the lowest id is the likeliest."""
    print("case: ties", flush=True)
    V = 20000
    x, tok, y, u, s = make(3, 4, V, "bf16", 5)
    took, count, chance = _one(lm, x, tok, x[:, :4].clone(),
                               torch.full((3, 4), 1 - 2.0 ** -24), s)
    assert count.tolist() == [4] * 3 and bool((chance == 1).all())
    flat = torch.zeros(1, 2, V)
    flat[0, 1, [9000, 17, 19999]] = 2.0
    took, count, _ = _one(lm, flat, torch.tensor([[0]]), temp=0.0)
    assert took.tolist() == [[0, 17]]
    took, count, _ = _one(lm, flat, torch.tensor([[1]]), temp=0.0)
    assert took.tolist() == [[0, -1]]
    # a flat row's draws lie where the running sum says
    for u_ in (0.0, 0.25, 0.7, 1 - 2.0 ** -24):
        took, *_ = _one(lm, flat[:, :1], torch.zeros(1, 0).long(),
                        s=torch.tensor([u_]))
        at = float(torch.tensor(u_).double()) * V
        assert int(took) in (int(at), max(int(at) - 1, 0))


def test_layouts(lm):
    """Views with strides of their own, odd starts, and vectors that have to
    be copied: as contiguous ones."""
    print("case: layouts", flush=True)
    x, tok, y, u, s = make(5, 3, 1003, "bf16", 6)
    big = torch.zeros(5, 4, 1003 + 7).bfloat16()
    big[..., 3:1006] = x
    turned = y.transpose(1, 2).contiguous().transpose(1, 2)
    major = x.transpose(0, 1).contiguous().transpose(0, 1)
    want = lm.verify_drafts(*(t.cuda() for t in (x, tok, y, u, s)))
    wide = torch.stack([tok, tok], -1).int().cuda()[..., 0]
    uu = torch.stack([u, u], 0).cuda()[1]
    for a, b in ((big.cuda()[..., 3:1006], turned.cuda()),
                 (major.cuda(), y.cuda())):
        assert not a.is_contiguous()
        got = lm.verify_drafts(a, wide, b, uu, s.cuda())
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    one = x[:, :1].cuda().expand(5, 4, 1003)
    a = lm.verify_drafts(one, tok.cuda(), None, u.cuda(), s.cuda())
    b = lm.verify_drafts(one.contiguous(), tok.cuda(), None, u.cuda(),
                         s.cuda())
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_distribution_of_what_is_emitted(lm):
    """With drafts drawn from q the first token emitted is distributed as p:
    the shares of q's drafts over a grid of both random numbers.  A grid of n
    midpoints misses the measure of an interval by at most 1 / n; of u there is
    one interval a draft (taken or not), 1 / 32, of s one a token, 1 / 512."""
    print("case: distribution", flush=True)
    V, n = 5, 512
    g = _gen(7)
    p, q = torch.randn(V, generator=g), torch.randn(V, generator=g)
    mid = (torch.arange(n) + 0.5) / n
    share = torch.zeros(V, dtype=torch.float64)
    qs = torch.softmax(q.double(), -1)
    x = p.cuda().expand(n, 2, V)
    for draft in range(V):
        tok = torch.full((n, 1), draft).cuda()
        for u in mid[::16]:
            got = lm.verify_drafts(x, tok, q.cuda().expand(n, 1, V),
                                   torch.full((n, 1), float(u)).cuda(),
                                   mid.cuda())
            first = got.tokens[:, 0].cpu()
            share += qs[draft] * torch.bincount(first, minlength=V) / n / 32
    off = (share - torch.softmax(p.double(), -1)).abs().max()
    assert float(off) <= 1 / 32 + 1 / 512, off


# --- sizes, streams, graphs ----------------------------------------------------

def test_offsets_past_32_bits(lm):
    print("case: offsets past 32 bits", flush=True)
    x, tok, y, u, s = (t.cuda() for t in make(2, 2, 70000, "bf16", 8))
    apart = 2 ** 31 + 5
    big = torch.zeros(apart + 3 * 70000, dtype=torch.bfloat16, device="cuda")
    far = big.as_strided((2, 3, 70000), (apart, 70000, 1))
    far.copy_(x)
    for q in (y, None):
        a = lm.verify_drafts(far, tok, q, u, s)
        b = lm.verify_drafts(x, tok, q, u, s)
        assert all(torch.equal(m, n) for m, n in zip(a, b))


def test_no_sequences_and_many(lm):
    print("case: none and many", flush=True)
    x, tok, y, u, s = (t.cuda() for t in make(3000, 1, 33, "f32", 9))
    got = lm.verify_drafts(x, tok, y, u, s)
    last = lm.verify_drafts(x[-2:], tok[-2:], y[-2:], u[-2:], s[-2:])
    assert all(torch.equal(a[-2:], b) for a, b in zip(got, last))
    none = lm.verify_drafts(x[:0], tok[:0], y[:0], u[:0], s[:0])
    assert [tuple(t.shape) for t in none] == [(0, 2), (0,), (0, 1)]


def test_streams_and_two_graphs(lm):
    print("case: streams and graphs", flush=True)
    cases = [[t.cuda() for t in make(6, 3, 30000, "bf16", i)] for i in (1, 2)]
    want = [lm.verify_drafts(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(4):
        for c, st in zip(cases, streams):
            with torch.cuda.stream(st):
                got.append(lm.verify_drafts(*c))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(out, want[i % 2]))
    graphs = []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[0]):
            out = lm.verify_drafts(*c)
        graphs.append((graph, out))
    for rep in range(4):
        for i in ((0, 1), (1, 0), (1, 1), (0, 0))[rep]:
            graph, out = graphs[i]
            for t in out:
                t.fill_(-7)
            lm.verify_drafts(*cases[1 - i])
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want[i])), rep

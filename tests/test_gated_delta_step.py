"""The gated delta rule on a pool of states (gdr_step.hip), and with the
verification of drafted tokens, against the recurrence in float64.

Tolerance, relative to an output's largest magnitude.  A token takes fp32
products of up to 128 terms, sqrt(128) 2^-24 = 7e-7 as signs differ, with the
old state twice, an exponential, 1e-7, and three roundings of the state, 2e-7:
1.7e-6, eight tokens 1.4e-5.  bf16 outputs are rounded once more, 2^-8.
"""

from __future__ import annotations

import pytest
import torch

from test_gated_delta import _gen, close, make, rule64

pytestmark = pytest.mark.gpu

STEP = 1.4e-5
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(scope="module")
def lm(hip_lib):
    import rwkv7m_amd
    return rwkv7m_amd


def want(x, states, rows, lengths, scale=None):
    """(o, states of the rows) with o 0 behind a row's length."""
    B, T, Hv, Dv = x[2].shape
    o = torch.zeros(B, T, Hv, Dv, dtype=torch.float64)
    ends = []
    for b in range(B):
        n = min(max(int(lengths[b]), 0), T)
        out, end = rule64(*(t[b:b + 1, :n] for t in x),
                          states[rows[b]:rows[b] + 1], scale)
        o[b, :n] = out[0]
        ends.append(end[0])
    return o, torch.stack(ends) if ends else states[:0].double()


def check(lm, x, pool, slots=None, lengths=None, scale=None, ids=torch.int64,
          place=lambda t: t.cuda()):
    B, T = x[0].shape[:2]
    rows = list(range(B)) if slots is None else slots
    n = [T] * B if lengths is None else lengths
    o, ends = want(x, pool, rows, n, scale)
    args = [place(t) for t in x]
    index = [None if t is None else torch.tensor(t, dtype=ids).cuda()
             for t in (lengths, slots)]
    state = pool.cuda()
    peeked = lm.gated_delta_step(*args, state, *index, scale=scale,
                                 update_state=False)
    assert torch.equal(state.cpu(), pool)
    got = lm.gated_delta_step(*args, state, *index, scale=scale)
    assert torch.equal(got, peeked) and got.dtype == x[2].dtype
    close("o", got, o, STEP)
    for b in range(B):
        assert not got[b, max(min(n[b], T), 0):].any()
    close("state", state[rows], ends, STEP)
    still = [i for i in range(len(pool)) if i not in rows or
             n[rows.index(i)] <= 0]
    assert torch.equal(state[still].cpu(), pool[still])


@pytest.mark.parametrize("T", [1, 2, 3, 8])
@pytest.mark.parametrize("Dk,Dv", [(8, 8), (64, 64), (72, 40), (128, 128),
                                   (40, 256), (128, 72)])
@pytest.mark.parametrize("dtype,gtype", [("bf16", "f32"), ("f32", "bf16")])
def test_sizes(lm, T, Dk, Dv, dtype, gtype):
    print("case: step", T, Dk, Dv, dtype, flush=True)
    x = make(3, T, 2, 4, Dk, Dv, dtype, gtype, seed=Dk + Dv + T)
    check(lm, x, torch.randn(3, 4, Dv, Dk, generator=_gen(T)))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("ids", [torch.int64, torch.int32])
def test_slots_and_lengths(lm, dtype, ids):
    print("case: slots", dtype, ids, flush=True)
    x = make(7, 5, 1, 3, 64, 64, dtype, seed=1)
    pool = torch.randn(11, 3, 64, 64, generator=_gen(2))
    check(lm, x, pool, [10, 0, 3, 7, 4, 9, 1], None, ids=ids)
    check(lm, x, pool, [10, 0, 3, 7, 4, 9, 1], [0, 1, 5, 9, -2, 4, 3],
          ids=ids)
    check(lm, x, pool[:7], None, [5, 4, 3, 2, 1, 0, 5], -0.5, ids=ids)


def test_slots_that_are_not_there(lm):
    """Padding, a slot past the pool, a slot given twice, and twice where the
    first has nothing to add."""
    print("case: bad slots", flush=True)
    x = [t.cuda() for t in make(6, 3, 1, 2, 64, 32, "bf16", seed=3)]
    pool = torch.randn(4, 2, 32, 64, generator=_gen(4)).cuda()
    slots = torch.tensor([2, -1, 4, 2, 0, 2 ** 40], device="cuda")
    state = pool.clone()
    o = lm.gated_delta_step(*x, state, slots=slots)
    alone = pool.clone()
    pick = torch.tensor([0, 4], device="cuda")
    right = lm.gated_delta_step(*(t[pick] for t in x), alone,
                                slots=slots[pick])
    assert torch.equal(o[pick], right) and torch.equal(state, alone)
    assert not o[1].any()
    for row in (2, 3, 5):
        assert o[row].isnan().all()
    assert torch.equal(state[[1, 3]], pool[[1, 3]])
    # read ahead, a slot may serve two rows
    ahead = lm.gated_delta_step(*x, pool, slots=slots, update_state=False)
    assert torch.equal(ahead[pick], right) and ahead[3].isfinite().all()
    # an earlier row of no tokens leaves the state to the later one
    lengths = torch.tensor([0, 3, 3, 2, 3, 0], device="cuda")
    state = pool.clone()
    o = lm.gated_delta_step(*x, state, lengths, slots)
    alone = pool.clone()
    one = lm.gated_delta_step(*(t[3:4] for t in x), alone, lengths[3:4],
                              slots[3:4])
    assert torch.equal(o[3:4], one) and torch.equal(state[2], alone[2])
    assert not o[0].any() and not o[5].any() and o[2].isnan().all()


def test_views_and_many_rows(lm):
    print("case: step views", flush=True)
    B, Hk, Hv, Dk, Dv = 300, 2, 4, 64, 64
    flat = torch.randn(B, 3, 2 * Hk * Dk + Hv * Dv, generator=_gen(5))
    flat = (0.1 * flat).bfloat16().cuda()
    q, k, v = flat.split((Hk * Dk, Hk * Dk, Hv * Dv), -1)
    q, k = (t.unflatten(-1, (Hk, Dk)) for t in (q, k))
    v = v.unflatten(-1, (Hv, Dv))
    gates = torch.rand(3, B, Hv, 2, generator=_gen(6)).cuda()
    g, beta = -gates.transpose(0, 1)[..., 0], gates.transpose(0, 1)[..., 1]
    a = torch.randn(B, Hv, Dv, Dk, generator=_gen(7)).cuda()
    b = a.clone()
    slots = torch.randperm(B, generator=_gen(8)).cuda()
    o = lm.gated_delta_step(q, k, v, g, beta, a, slots=slots)
    p = lm.gated_delta_step(*(t.contiguous() for t in (q, k, v, g, beta)), b,
                            slots=slots)
    assert torch.equal(o, p) and torch.equal(a, b)
    # a row's result is its own, whatever else is in the call
    c = torch.randn(B, Hv, Dv, Dk, generator=_gen(7)).cuda()
    one = lm.gated_delta_step(*(t[7:8] for t in (q, k, v, g, beta)), c,
                              slots=slots[7:8])
    assert torch.equal(one, o[7:8])
    assert torch.equal(c[slots[7]], a[slots[7]])


def test_step_goes_on_from_the_rule(lm):
    """A prompt by gated_delta_rule, tokens by gated_delta_step, against both
    in one rule: the state is the same thing to both."""
    print("case: prompt, then steps", flush=True)
    x = make(2, 90, 1, 2, 64, 64, "f32", seed=9)
    whole, end = rule64(*x)
    x = [t.cuda() for t in x]
    _, state = lm.gated_delta_rule(*(t[:, :82] for t in x))
    outs = [lm.gated_delta_step(*(t[:, i:i + 1] for t in x), state)
            for i in range(82, 90)]
    # (the rule's NARROW, 1.5e-5, and the steps')
    close("o", torch.cat(outs, 1), whole[:, 82:], 1.5e-5 + STEP)
    close("state", state, end, 1.5e-5 + STEP)


@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("captured", [False, True])
def test_drafts_are_read_verified_and_taken(lm, temperature, captured):
    """What serving does with a block of drafted tokens: the layer reads it
    ahead, the head's logits are verified, and the tokens that hold go into
    the states.  The states are those of the accepted tokens one at a time,
    the outputs of the first call those of a plain decode, eagerly and as one
    graph replayed over several blocks."""
    print("case: speculative decode", temperature, captured, flush=True)
    B, K, H, D, V = 5, 3, 2, 64, 400
    g = _gen(30)
    head = (0.4 * torch.randn(V, H * D, generator=g)).cuda()
    table = [t for t in make(V, 1, H, H, D, D, "f32", seed=31)]
    table = [t[:, 0].cuda() for t in table]  # a token's vectors and gates
    slots = torch.tensor([4, 2, 6, 0, 3], device="cuda")
    pool = torch.randn(7, H, D, D, generator=g).cuda()
    last = torch.randint(0, V, (B,), generator=g).cuda()
    drafts = torch.zeros(B, K, dtype=torch.int64, device="cuda")
    u, s = torch.zeros(B, K, device="cuda"), torch.zeros(B, device="cuda")
    state = pool.clone()

    def block():
        tokens = torch.cat([last[:, None], drafts], 1)
        x = [t[tokens] for t in table]
        o = lm.gated_delta_step(*x, state, slots=slots, update_state=False)
        logits = (o.flatten(2)[:, :, None] * head).sum(-1)
        got = lm.verify_drafts(logits, drafts, None, u, s,
                               temperature=temperature)
        lm.gated_delta_step(*x, state, got.accepted + 1, slots)
        return tokens, o, logits, got

    def fill(i):
        r = _gen(40 + i)
        drafts.copy_(torch.randint(0, V, (B, K), generator=r))
        u.copy_(torch.rand(B, K, generator=r))
        s.copy_(torch.rand(B, generator=r))
        # likely drafts for some rows, so that some are taken
        probe = state.clone()
        word = last.clone()
        for j in range(K):
            x = [t[word][:, None] for t in table]
            o = lm.gated_delta_step(*x, probe, slots=slots)
            word = (o.flatten(2)[:, 0] @ head.T).argmax(-1)
            drafts[::2, j] = word[::2]
        u[::2] *= 1e-3

    graph = None
    if captured:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            static = block()
        state.copy_(pool)
    taken = 0
    for i in range(4):
        fill(i)
        before = state.clone()
        torch.cuda.synchronize()
        if graph is None:
            tokens, o, logits, got = block()
        else:
            graph.replay()
            tokens, o, logits, got = static
        torch.cuda.synchronize()
        # plain decode over the tokens that hold
        plain = before.clone()
        for j in range(K + 1):
            x = [t[tokens[:, j]][:, None] for t in table]
            live = (got.accepted >= j).long()
            one = lm.gated_delta_step(*x, plain, live, slots)
            rows = live.bool()
            close("o", one[rows, 0], o[rows, j].double().cpu(), STEP)
        close("state", plain, state.double().cpu(), STEP)
        p = torch.softmax(logits.double(), -1)
        for b in range(B):
            m = int(got.accepted[b])
            for j in range(K):
                at = int(drafts[b, j])
                ok = (at == int(logits[b, j].argmax()) if temperature == 0
                      else float(u[b, j].double()) < float(p[b, j, at]))
                assert ok if j < m else (ok is False if j == m else True)
            assert torch.equal(got.tokens[b, :m], drafts[b, :m])
            assert 0 <= int(got.tokens[b, m]) < V
            assert bool((got.tokens[b, m + 1:] == -1).all())
            last[b] = got.tokens[b, m]
        taken += int(got.accepted.sum())
    assert 4 * K <= taken < 4 * B * K  # (both kinds of rows were there)
    assert torch.equal(state[[1, 5]], pool[[1, 5]])


# --- streams and graphs --------------------------------------------------------

def _train(lm, leaves, do, ds):
    o, end = lm.gated_delta_rule(*leaves)
    return [o, end, *torch.autograd.grad([o, end], leaves, [do, ds])]


def _leaves(seed, Hv=2):
    x = [t.cuda() for t in make(2, 130, 1, Hv, 64, 64, "bf16", seed=seed)]
    x.append(torch.randn(2, Hv, 64, 64, generator=_gen(seed)).cuda())
    do = torch.randn(2, 130, Hv, 64, generator=_gen(seed)).bfloat16().cuda()
    return [t.requires_grad_() for t in x], do, torch.randn(
        2, Hv, 64, 64, generator=_gen(seed + 1)).cuda()


def test_side_stream_and_two_graphs(lm):
    """Forward and backward on another stream, and two captured graphs (of
    several workspaces each), replayed in turn with eager work between."""
    print("case: training graphs", flush=True)
    cases = [_leaves(1), _leaves(2, 3)]
    want = [_train(lm, *c) for c in cases]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [_train(lm, *c) for c in cases]
    side.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    del got
    graphs = []
    for leaves, do, ds in cases:
        own = [t.detach().clone().requires_grad_() for t in leaves]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = [t.detach() for t in _train(lm, own, do, ds)]
        graphs.append((graph, out, own))
    for rep in range(4):
        for i in ((0, 1), (1, 0), (1, 1), (0, 0))[rep]:
            graph, out, _ = graphs[i]
            for t in out:
                t.fill_(-7)
            _train(lm, *cases[1 - i])
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want[i]):
                assert torch.equal(a, b), f"replay {rep}"


def test_two_streams_at_once(lm):
    print("case: two streams", flush=True)
    cases = [_leaves(3), _leaves(4, 3)]
    want = [_train(lm, *c) for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(_train(lm, *c))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(out, want[i % 2]))


def test_inference_mode_and_two_calls_on_one_pool(lm):
    """States made inside and outside of inference mode, and two streams at
    work on different slots of one pool."""
    print("case: inference mode", flush=True)
    x = [t.cuda() for t in make(4, 2, 1, 2, 64, 64, "bf16", seed=15)]
    pool = torch.randn(8, 2, 64, 64, generator=_gen(1)).cuda()
    slots = torch.tensor([5, 0, 7, 2], device="cuda")
    want = pool.clone()
    o = lm.gated_delta_step(*x, want, slots=slots)
    outer = pool.clone()
    with torch.inference_mode():
        inner = pool.clone()
        for state in (inner, outer):
            assert torch.equal(lm.gated_delta_step(*x, state, slots=slots), o)
            assert torch.equal(state, want)
        a, end = lm.gated_delta_rule(*x, pool[slots])
        tok = torch.zeros(4, 1, dtype=torch.int64, device="cuda")
        lm.verify_drafts(a.float().flatten(2), tok, temperature=0.0)
    state = pool.clone()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            outs.append(lm.gated_delta_step(
                *(t[2 * i:2 * i + 2] for t in x), state,
                slots=slots[2 * i:2 * i + 2]))
    torch.cuda.synchronize()
    assert torch.equal(torch.cat(outs), o) and torch.equal(state, want)

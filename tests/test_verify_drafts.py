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

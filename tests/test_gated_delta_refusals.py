"""What the gated delta rule, its step and the verification of drafted tokens
refuse: wrong shapes, types and sizes before anything reaches the device (these
run without a GPU; no valid request is made)."""

from __future__ import annotations

import ctypes
import os

import pytest
import torch

from rwkv7m_amd import gated_delta_rule, gated_delta_step, verify_drafts

P = 4096  # an address: nothing is read before every check has passed


@pytest.fixture(scope="module")
def lib():
    from rwkv7m_amd import _build
    from rwkv7m_amd.kernels import wkv_hip
    if not os.path.exists(wkv_hip.LIB_PATH):
        _build.build()
    return wkv_hip.load_library()


class Inputs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("dtype", "g_dtype", "beta_dtype")] \
        + [(n, ctypes.c_int64) for n in ("B", "T", "Hk", "Hv", "Dk", "Dv")] \
        + [(n, ctypes.c_void_p) for n in ("q", "k", "v", "g", "beta")] \
        + [(n + "_stride", ctypes.c_int64 * 3)
           for n in ("q", "k", "v", "g", "beta")] \
        + [("scale", ctypes.c_double)]


def _inputs(**kw):
    x = Inputs(dtype=1, g_dtype=0, beta_dtype=0, B=2, T=5, Hk=2, Hv=4, Dk=64,
               Dv=32, q=P, k=P, v=P, g=P, beta=P, scale=0.125)
    x.q_stride[:] = x.k_stride[:] = (5 * 128, 128, 64)
    x.v_stride[:] = (5 * 128, 128, 32)
    x.g_stride[:] = x.beta_stride[:] = (20, 4, 1)
    for name, value in kw.items():
        if name.endswith("_stride"):
            getattr(x, name)[:] = value
        else:
            setattr(x, name, value)
    return x


def _refused(lib, rc, code, words):
    assert rc == code and words in lib.rwkv7m_last_error().decode(), (
        rc, lib.rwkv7m_last_error())


BAD_INPUTS = (
    (dict(dtype=5), 1, "q, k and v must be bfloat16 or float32"),
    (dict(g_dtype=2), 1, "g must be"), (dict(beta_dtype=-1), 1, "beta must"),
    (dict(B=-1), 1, "negative"), (dict(T=-1), 1, "negative"),
    (dict(Hk=0), 1, "multiple of Hk"), (dict(Hk=3), 1, "multiple of Hk"),
    (dict(Dk=0), 2, "head sizes"), (dict(Dk=12), 2, "head sizes"),
    (dict(Dk=136), 2, "head sizes"), (dict(Dv=264), 2, "head sizes"),
    (dict(scale=float("nan")), 1, "scale"),
    (dict(scale=float("inf")), 1, "scale"),
    (dict(B=1 << 30), 1, "too large"), (dict(T=1 << 41), 1, "too large"),
    (dict(T=1 << 30), 1, "too large"), (dict(B=1 << 20), 1, "too large"),
    (dict(q=None), 1, "q is NULL"), (dict(k=None), 1, "k is NULL"),
    (dict(v=None), 1, "v is NULL"), (dict(g=None), 1, "g is NULL"),
    (dict(beta=None), 1, "beta is NULL"), (dict(q=P + 8), 1, "16-byte"),
    (dict(g=P + 2), 1, "4-byte"),
    (dict(k_stride=(640, -128, 64)), 1, "negative stride"),
    (dict(q_stride=(640, 132, 64)), 1, "rows are not 16-byte aligned"),
    (dict(g_stride=(1 << 62, 4, 1)), 1, "too large"))


def test_rule_refuses(lib):
    def call(x, s0=None, o=P, end=P, saved=None, ws=P, size=1 << 30):
        return lib.rwkv7m_gated_delta_rule(
            None if x is None else ctypes.byref(x), s0, o, end, saved, ws,
            size, None)

    _refused(lib, call(None), 1, "inputs is NULL")
    for kw, code, words in BAD_INPUTS + ((dict(v=P + 8), 1, "16-byte"),):
        _refused(lib, call(_inputs(**kw)), code, words)
        assert "rwkv7m_gated_delta_rule:" in lib.rwkv7m_last_error().decode()
    need = lib.rwkv7m_gated_delta_workspace_bytes(ctypes.byref(_inputs()), 0)
    assert need > 0
    for kw, words in ((dict(o=None), "o is NULL"),
                      (dict(o=P + 2), "o is not 16-byte"),
                      (dict(s0=P + 4), "initial_state is not"),
                      (dict(end=P + 8), "final_state is not"),
                      (dict(saved=P + 4), "saved is not"),
                      (dict(size=need - 1), "workspace holds"),
                      (dict(ws=None), "workspace is NULL")):
        _refused(lib, call(_inputs(), **kw), 1, words)
    assert call(_inputs(B=0), o=None, ws=None, size=0) == 0
    assert call(_inputs(T=0), o=None, end=None, ws=None, size=0) == 0
    for bad in (dict(Dk=4), dict(B=-1), dict(T=1 << 41)):
        x = ctypes.byref(_inputs(**bad))
        assert lib.rwkv7m_gated_delta_workspace_bytes(x, 1) == -1
        assert lib.rwkv7m_gated_delta_saved_floats(x) == -1


def test_rule_backward_refuses(lib):
    def call(x, do=P, stride=(640, 128, 32), ds=None, saved=P, dq=P, dk=P,
             dv=P, dg=P, db=P, d0=None, ws=P, size=1 << 30):
        st = None if stride is None else (ctypes.c_int64 * 3)(*stride)
        return lib.rwkv7m_gated_delta_rule_backward(
            ctypes.byref(x), do, st, ds, saved, dq, dk, dv, dg, db, d0, ws,
            size, None)

    for kw, code, words in BAD_INPUTS:
        _refused(lib, call(_inputs(**kw)), code, words)
    need = lib.rwkv7m_gated_delta_workspace_bytes(ctypes.byref(_inputs()), 1)
    for kw, words in ((dict(do=None), "d_o is NULL"),
                      (dict(stride=None), "d_o_stride is NULL"),
                      (dict(stride=(640, 130, 32)), "aligned"),
                      (dict(stride=(640, -1, 32)), "negative stride"),
                      (dict(saved=None), "saved is NULL"),
                      (dict(dq=None), "dq is NULL"),
                      (dict(dk=P + 8), "dk is not"),
                      (dict(dv=None), "dv is NULL"),
                      (dict(dg=None), "dg is NULL"),
                      (dict(db=P + 1), "dbeta is not"),
                      (dict(ds=P + 4), "d_final_state is not"),
                      (dict(d0=P + 4), "d_initial_state is not"),
                      (dict(size=need - 1), "workspace holds"),
                      (dict(ws=None), "workspace is NULL")):
        _refused(lib, call(_inputs(), **kw), 1, words)


def test_step_refuses(lib):
    def call(x, pool=2, state=P, slots=None, lengths=None, update=1, o=P):
        return lib.rwkv7m_gated_delta_step(
            ctypes.byref(x), pool, state, slots, lengths, update, o, None)

    for kw, code, words in BAD_INPUTS:
        if "B" not in kw:
            _refused(lib, call(_inputs(**kw)), code, words)
    for kw, words in ((dict(pool=1), "a pool of 1 states for B=2"),
                      (dict(pool=-1, slots=P), "a pool of -1"),
                      (dict(pool=1 << 45, slots=P), "too large"),
                      (dict(slots=P + 4), "slots is not 8-byte"),
                      (dict(lengths=P + 4), "lengths is not 8-byte"),
                      (dict(state=None), "state is NULL"),
                      (dict(state=P + 4), "state is not 16-byte"),
                      (dict(o=None), "o is NULL")):
        _refused(lib, call(_inputs(), **kw), 1, words)
    assert call(_inputs(B=0), pool=0, state=None, o=None) == 0
    assert call(_inputs(T=0), o=None) == 0


def test_verification_refuses(lib):
    need = lib.rwkv7m_verify_drafts_workspace_bytes(2, 3, 50)
    assert need > 0

    def call(dtype=1, B=2, K=3, V=50, x=P, os_=200, is_=50, y=P, ys=(150, 50),
             tok=P, u=P, s=P, n=None, temp=1.0, out=P, took=P, chance=P,
             ws=P, size=need):
        return lib.rwkv7m_verify_drafts(
            dtype, B, K, V, os_, is_, x, *ys, y, tok, u, s, n, temp, out, took,
            chance, ws, size, None)

    for kw, code, words in (
            (dict(dtype=4), 1, "logits must be"), (dict(B=-1), 1, "negative"),
            (dict(K=-1), 1, "K=-1"), (dict(K=65), 2, "not supported"),
            (dict(V=0), 1, "element"), (dict(is_=-1), 1, "negative"),
            (dict(ys=(-1, 50)), 1, "negative"),
            (dict(V=1 << 31), 1, "too large"),
            (dict(B=1 << 26), 1, "too large"),
            (dict(temp=-1.0), 1, "temperature"),
            (dict(temp=1e-40), 1, "temperature"),
            (dict(temp=float("nan")), 1, "temperature"),
            (dict(temp=float("inf")), 1, "temperature"),
            (dict(x=None), 1, "logits is NULL"),
            (dict(x=P + 1), 1, "logits is not"),
            (dict(y=P + 1), 1, "draft logits is not"),
            (dict(tok=None), 1, "tokens is NULL"),
            (dict(tok=P + 4), 1, "tokens is not 8-byte"),
            (dict(u=None), 1, "accept is NULL"),
            (dict(s=None), 1, "sample is NULL"),
            (dict(n=P + 4), 1, "draft_lengths is not"),
            (dict(out=None), 1, "out is NULL"),
            (dict(took=None), 1, "accepted is NULL"),
            (dict(chance=None), 1, "chances is NULL"),
            (dict(ws=None), 1, "workspace is NULL"),
            (dict(size=need - 1), 1, "workspace holds")):
        _refused(lib, call(**kw), code, words)
        assert "rwkv7m_verify_drafts:" in lib.rwkv7m_last_error().decode()
    assert call(B=0, x=None, y=None, tok=None, u=None, s=None, out=None,
                took=None, chance=None, ws=None, size=0) == 0
    for bad in ((-1, 3, 50), (2, 65, 50), (2, 3, 0), (1 << 25, 3, 50)):
        assert lib.rwkv7m_verify_drafts_workspace_bytes(*bad) == -1


def _args(B=2, T=3, Hk=1, Hv=2, Dk=16, Dv=8, dtype=torch.float32):
    return [torch.zeros(B, T, Hk, Dk, dtype=dtype),
            torch.zeros(B, T, Hk, Dk, dtype=dtype),
            torch.zeros(B, T, Hv, Dv, dtype=dtype), torch.zeros(B, T, Hv),
            torch.zeros(B, T, Hv)]


def _but(**kw):
    names = ("q", "k", "v", "g", "beta")
    return [kw.get(n, t) for n, t in zip(names, _args())]


@pytest.mark.parametrize("step", [False, True])
def test_python_calls_refuse(step):
    q, k, v, g, beta = _args()
    state = torch.zeros(2, 2, 8, 16)

    def call(x):
        return gated_delta_step(*x, state) if step else gated_delta_rule(*x)

    for kind, words, kw in (
            (RuntimeError, "GPU tensors", {}),
            (TypeError, "q must be bfloat16 or float32", dict(q=q.half())),
            (TypeError, "share one dtype", dict(k=k.bfloat16())),
            (TypeError, "share one dtype", dict(v=v.bfloat16())),
            (TypeError, "g must be", dict(g=g.double())),
            (TypeError, "beta must be", dict(beta=beta.int())),
            (ValueError, "q must have shape", dict(q=q[0])),
            (ValueError, "k must have shape", dict(k=k[:, :2])),
            (ValueError, "v must have shape", dict(v=v[:1])),
            (ValueError, "v must have shape", dict(v=v[0])),
            (ValueError, "g must have shape", dict(g=g[..., :1])),
            (ValueError, "beta must have shape", dict(beta=beta[..., None])),
            (ValueError, "multiple of q's", dict(q=q.expand(2, 3, 4, 16),
                                                 k=k.expand(2, 3, 4, 16))),
            (ValueError, "multiples of 8", dict(q=q[..., :12],
                                                k=k[..., :12])),
            (ValueError, "multiples of 8", dict(v=v[..., :4]))):
        with pytest.raises(kind, match=words):
            call(_but(**kw))


def test_python_step_refuses():
    x = _args()
    state, ids = torch.zeros(4, 2, 8, 16), torch.zeros(2, dtype=torch.int64)
    for kind, words, s, kw in (
            (ValueError, "state must have shape", state[0], {}),
            (ValueError, "state must have shape", state.mT, {}),
            (TypeError, "state must be float32", state.double(), {}),
            (ValueError, "contiguous", state[:, :, :, :8].repeat(
                1, 1, 1, 4)[..., ::2], dict(slots=ids)),
            (ValueError, "a state for each", state, {}),
            (ValueError, "slots must have shape", state,
             dict(slots=ids[:1])),
            (TypeError, "slots must be", state, dict(slots=ids.float())),
            (ValueError, "lengths must have shape", state,
             dict(lengths=ids[:, None], slots=ids)),
            (TypeError, "lengths must be", state,
             dict(lengths=ids.short(), slots=ids)),
            (RuntimeError, "GPU tensors", state, dict(slots=ids)),
            (RuntimeError, "no gradient", state.clone().requires_grad_(),
             dict(slots=ids))):
        with pytest.raises(kind, match=words):
            gated_delta_step(*x, s, **kw)


def test_python_verification_refuses():
    x, tok = torch.zeros(2, 4, 50), torch.zeros(2, 3, dtype=torch.int64)
    u, s = torch.zeros(2, 3), torch.zeros(2)
    y = x[:, :3]
    for kind, words, call in (
            (RuntimeError, "GPU tensors",
             lambda: verify_drafts(x, tok, y, u, s)),
            (TypeError, "logits must be",
             lambda: verify_drafts(x.half(), tok, None, u, s)),
            (ValueError, "logits must have shape",
             lambda: verify_drafts(x[0], tok, None, u, s)),
            (ValueError, "logits must have shape",
             lambda: verify_drafts(x[..., :0], tok, None, u, s)),
            (ValueError, "draft_tokens must have shape",
             lambda: verify_drafts(x, tok[:, :2], None, u, s)),
            (TypeError, "draft_tokens must be",
             lambda: verify_drafts(x, tok.float(), None, u, s)),
            (ValueError, "draft_logits must have shape",
             lambda: verify_drafts(x, tok, x, u, s)),
            (TypeError, "share one dtype",
             lambda: verify_drafts(x, tok, y.bfloat16(), u, s)),
            (ValueError, "draft_lengths must have shape",
             lambda: verify_drafts(x, tok, y, u, s, tok)),
            (TypeError, "draft_lengths must be",
             lambda: verify_drafts(x, tok, y, u, s, s)),
            (ValueError, "at most 64",
             lambda: verify_drafts(torch.zeros(1, 66, 5),
                                   torch.zeros(1, 65).long(), None,
                                   torch.zeros(1, 65), s[:1]))):
        with pytest.raises(kind, match=words):
            call()


@pytest.mark.gpu
def test_calls_on_the_gpu_refuse(hip_lib):
    print("case: refusals on the GPU", flush=True)
    x = [t.cuda() for t in _args()]
    state = torch.zeros(2, 2, 8, 16, device="cuda")
    odd = torch.zeros(2 * 2 * 8 * 16 + 1, device="cuda")[1:].view(2, 2, 8, 16)
    logits = torch.zeros(2, 4, 50, device="cuda")
    tok = torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    u, s = torch.zeros(2, 3, device="cuda"), torch.zeros(2, device="cuda")
    for kind, words, call in (
            (RuntimeError, "GPU tensors",
             lambda: gated_delta_rule(*x[:4], x[4].cpu())),
            (ValueError, "initial_state must have shape",
             lambda: gated_delta_rule(*x, state[0])),
            (TypeError, "initial_state must be",
             lambda: gated_delta_rule(*x, state.double())),
            (RuntimeError, "GPU tensors",
             lambda: gated_delta_rule(*x, state.cpu())),
            (RuntimeError, "scale is not finite",
             lambda: gated_delta_rule(*x, scale=float("inf"))),
            (RuntimeError, "GPU tensors",
             lambda: gated_delta_step(*x, state.cpu())),
            (RuntimeError, "state is not 16-byte",
             lambda: gated_delta_step(*x, odd)),
            (RuntimeError, "no gradient",
             lambda: gated_delta_step(*x, state.clone().requires_grad_())),
            (RuntimeError, "GPU tensors",
             lambda: gated_delta_step(*x, state, tok[:, 0].cpu())),
            (RuntimeError, "GPU tensors",
             lambda: verify_drafts(logits, tok.cpu(), None, u, s)),
            (ValueError, "accept_uniforms",
             lambda: verify_drafts(logits, tok, None, None, s)),
            (ValueError, "sample_uniforms",
             lambda: verify_drafts(logits, tok, None, u)),
            (ValueError, "accept_uniforms must have shape",
             lambda: verify_drafts(logits, tok, None, s, s)),
            (TypeError, "sample_uniforms must be",
             lambda: verify_drafts(logits, tok, None, u, s.double())),
            (RuntimeError, "temperature",
             lambda: verify_drafts(logits, tok, None, u, s,
                                   temperature=-1.0))):
        with pytest.raises(kind, match=words):
            call()

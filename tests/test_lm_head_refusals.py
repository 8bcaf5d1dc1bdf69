"""What the operators around a language model's head refuse: wrong shapes,
types and sizes before anything reaches the device (these run without a GPU;
no valid request is made)."""

from __future__ import annotations

import os

import pytest
import torch

from rwkv7m_amd import distill_loss, layer_norm, token_logprobs


@pytest.fixture(scope="module")
def lib():
    from rwkv7m_amd import _build
    from rwkv7m_amd.kernels import wkv_hip
    if not os.path.exists(wkv_hip.LIB_PATH):
        _build.build()
    return wkv_hip.load_library()


def _refused(lib, rc, code, words):
    assert rc == code and words in lib.rwkv7m_last_error().decode(), (
        rc, lib.rwkv7m_last_error())


def test_c_entry_points_refuse(lib):
    P = 4096  # an address: nothing is read before every check has passed
    norm = lib.rwkv7m_layer_norm

    def n(dtype=0, pdtype=0, outer=1, inner=2, C=8, os_=0, is_=8, x=P, w=P,
          b=P, eps=1e-5, y=P, mean=None, rstd=None):
        return norm(dtype, pdtype, outer, inner, C, os_, is_, x, w, b, eps, y,
                    mean, rstd, None)

    for kw, code, words in (
            (dict(dtype=7), 1, "x must be bfloat16 or float32"),
            (dict(pdtype=2), 1, "weight and bias must be"),
            (dict(C=0), 1, "at least one element"),
            (dict(inner=-1), 1, "negative"),
            (dict(is_=-8), 1, "negative"),
            (dict(C=1 << 40), 1, "too large"),
            (dict(outer=1 << 39, inner=1 << 39), 1, "too large"),
            (dict(is_=1 << 60), 1, "too large"),
            (dict(eps=-1.0), 1, "eps"), (dict(eps=float("nan")), 1, "eps"),
            (dict(x=None), 1, "x is NULL"), (dict(y=None), 1, "y is NULL"),
            (dict(x=P + 1), 1, "aligned"), (dict(w=P + 2), 1, "aligned"),
            (dict(mean=P), 1, "go together")):
        _refused(lib, n(**kw), code, words)
        assert "rwkv7m_layer_norm:" in lib.rwkv7m_last_error().decode()
    assert n(inner=0, x=None, y=None) == 0
    assert lib.rwkv7m_layer_norm_workspace_floats(-1, 8) == -1
    assert lib.rwkv7m_layer_norm_workspace_floats(3, 0) == -1
    floats = lib.rwkv7m_layer_norm_workspace_floats(100, 64)
    assert floats >= 2 * 64

    def nb(x=P, mean=P, dy=P, dx=P, dw=P, db=P, ws=P, floats=floats):
        return lib.rwkv7m_layer_norm_backward(
            1, 0, 1, 100, 64, 0, 64, x, P, mean, P, dy, dx, dw, db, ws,
            floats, None)

    for kw, words in ((dict(floats=floats - 1), "workspace holds"),
                      (dict(ws=None), "workspace is NULL"),
                      (dict(mean=None), "mean is NULL"),
                      (dict(dy=None), "dy is NULL"),
                      (dict(dx=P + 1), "dx is not 2-byte aligned"),
                      (dict(dw=P + 2), "dweight is not 4-byte aligned")):
        _refused(lib, nb(**kw), 1, words)

    def s(dtype=1, V=50, logits=P, tokens=P, k=2, temp=1.0, lp=P, ent=P,
          ids=P, top=P):
        return lib.rwkv7m_token_logprobs(dtype, 1, 3, V, 0, V, logits, tokens,
                                         k, temp, lp, ent, ids, top, None,
                                         None)

    for kw, code, words in (
            (dict(dtype=3), 1, "logits must be"), (dict(V=0), 1, "element"),
            (dict(k=51), 1, "top_k=51"), (dict(k=-1), 1, "top_k"),
            (dict(V=500, k=65), 2, "not supported"),
            (dict(temp=0.0), 1, "temperature"),
            (dict(temp=-1.0), 1, "temperature"),
            (dict(temp=float("nan")), 1, "temperature"),
            (dict(temp=float("inf")), 1, "temperature"),
            (dict(logits=P + 1), 1, "aligned"),
            (dict(tokens=None), 1, "tokens is NULL"),
            (dict(tokens=P + 4), 1, "8-byte"), (dict(lp=None), 1, "logprobs"),
            (dict(ids=None), 1, "top_ids"), (dict(top=None), 1, "top_logp")):
        _refused(lib, s(**kw), code, words)
    bwd = lib.rwkv7m_token_logprobs_backward
    _refused(lib, bwd(1, 1, 3, 50, 0, 50, P, P, 1.0, None, P, P, P, P, None),
             1, "stats is NULL")
    _refused(lib, bwd(1, 1, 3, 50, 0, 50, P, P, 1.0, P, P, P, P, None, None),
             1, "dlogits is NULL")

    def d(V=50, K=4, logits=P, ids=P, teacher=P, tdtype=0, w=None, temp=1.0,
          loss=P, rows=P, dl=P):
        return lib.rwkv7m_distill_loss(1, tdtype, 1, 3, V, 0, V, K, logits,
                                       ids, teacher, w, temp, loss, rows, dl,
                                       None)

    for kw, code, words in (
            (dict(K=257), 2, "not supported"), (dict(K=-1), 1, "K=-1"),
            (dict(tdtype=9), 1, "teacher logits must be"),
            (dict(ids=None), 1, "teacher_ids is NULL"),
            (dict(teacher=None), 1, "teacher_logits is NULL"),
            (dict(temp=0.0), 1, "temperature"), (dict(loss=None), 1, "loss"),
            (dict(rows=None), 1, "row_losses is NULL"),
            (dict(w=P + 1), 1, "weight is not"),
            (dict(dl=P + 1), 1, "dlogits is not")):
        _refused(lib, d(**kw), code, words)
    _refused(lib, lib.rwkv7m_distill_loss_backward(
        1, 0, 1, 3, 50, 0, 50, 4, P, P, P, None, 1.0, None, 0, P, None), 1,
        "scale is NULL")


def test_python_calls_refuse():
    x, i = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64)
    w = torch.zeros(8)
    cases = [
        (RuntimeError, "GPU tensors", lambda: layer_norm(x)),
        (TypeError, "bfloat16 or float32", lambda: layer_norm(x.double())),
        (TypeError, "bfloat16 or float32", lambda: layer_norm(x, w.half())),
        (ValueError, "weight must have shape",
         lambda: layer_norm(x, w[:7])),
        (ValueError, "bias must have shape",
         lambda: layer_norm(x, w, w.view(1, 8))),
        (TypeError, "share one dtype",
         lambda: layer_norm(x, w, w.bfloat16())),
        (ValueError, "at least one element", lambda: layer_norm(x[:, :0])),
        (ValueError, "at least one element",
         lambda: layer_norm(torch.tensor(1.0))),
        (RuntimeError, "GPU tensors", lambda: token_logprobs(x, i)),
        (TypeError, "bfloat16 or float32",
         lambda: token_logprobs(x.half(), i)),
        (ValueError, "tokens must have shape",
         lambda: token_logprobs(x, i[:2])),
        (TypeError, "int64 or int32",
         lambda: token_logprobs(x, i.float())),
        (ValueError, "teacher_logits must have shape",
         lambda: distill_loss(x, torch.zeros(2, 4).long(),
                              torch.zeros(2, 4))),
        (ValueError, "teacher_ids must have shape",
         lambda: distill_loss(x, torch.zeros(3, 5).long(),
                              torch.zeros(3, 4))),
        (TypeError, "int64 or int32",
         lambda: distill_loss(x, torch.zeros(3, 4), torch.zeros(3, 4))),
        (TypeError, "teacher_logits must be",
         lambda: distill_loss(x, torch.zeros(3, 4).long(),
                              torch.zeros(3, 4).half())),
        (ValueError, "at most 256",
         lambda: distill_loss(x, torch.zeros(3, 257).long(),
                              torch.zeros(3, 257))),
        (ValueError, "weight must have shape",
         lambda: distill_loss(x, torch.zeros(3, 4).long(),
                              torch.zeros(3, 4), w)),
        (RuntimeError, "GPU tensors",
         lambda: distill_loss(x, torch.zeros(3, 4).long(),
                              torch.zeros(3, 4))),
    ]
    for kind, words, call in cases:
        with pytest.raises(kind, match=words):
            call()


@pytest.mark.gpu
def test_calls_on_the_gpu_refuse(hip_lib):
    print("case: refusals on the GPU", flush=True)
    x = torch.zeros(3, 80, device="cuda")
    i = torch.zeros(3, dtype=torch.int64, device="cuda")
    t = torch.zeros(3, 4, device="cuda")
    for kind, words, call in (
            (RuntimeError, "GPU tensors", lambda: token_logprobs(x, i.cpu())),
            (ValueError, "top_k", lambda: token_logprobs(x, i, top_k=65)),
            (ValueError, "top_k", lambda: token_logprobs(x, i, top_k=-1)),
            (ValueError, "top_k",
             lambda: token_logprobs(x[:, :5], i, top_k=6)),
            (RuntimeError, "temperature",
             lambda: token_logprobs(x, i, temperature=0.0)),
            (RuntimeError, "eps", lambda: layer_norm(x, eps=-1.0)),
            (RuntimeError, "temperature",
             lambda: distill_loss(x, t.long(), t, temperature=-2.0)),
            (RuntimeError, "GPU tensors",
             lambda: distill_loss(x, t.long(), t, torch.ones(3)))):
        with pytest.raises(kind, match=words):
            call()


def _with_tangents(x, i, t, w, c):
    """(name, call on inputs of which one has a tangent)"""
    dual = torch.autograd.forward_ad.make_dual

    def d(v):
        return dual(v, torch.ones_like(v))

    yield "layer_norm", lambda: layer_norm(d(x), c, c)
    yield "layer_norm", lambda: layer_norm(x, d(c), c)
    yield "layer_norm", lambda: layer_norm(x, c, d(c))
    yield "layer_norm", lambda: layer_norm(d(x))
    yield "token_logprobs", lambda: token_logprobs(d(x), i, top_k=2)
    yield "distill_loss", lambda: distill_loss(d(x), t.long(), t)
    yield "distill_loss", lambda: distill_loss(x, t.long(), d(t))
    yield "distill_loss", lambda: distill_loss(x, t.long(), t, d(w))


def _refuses_tangents(device):
    x, c = torch.zeros(3, 8, device=device), torch.ones(8, device=device)
    i = torch.zeros(3, dtype=torch.int64, device=device)
    t, w = torch.zeros(3, 4, device=device), torch.ones(3, device=device)
    words = " supports reverse-mode differentiation only"
    with torch.autograd.forward_ad.dual_level():
        for leaf in (x, x.clone().requires_grad_()):
            for name, call in _with_tangents(leaf, i, t, w, c):
                for grad in (torch.enable_grad, torch.no_grad):
                    with grad(), pytest.raises(TypeError, match=name + words):
                        call()
    for name, f in (
            ("layer_norm", layer_norm),
            ("token_logprobs", lambda v: token_logprobs(v, i).logprobs),
            ("distill_loss", lambda v: distill_loss(v, t.long(), t).loss)):
        with pytest.raises(TypeError, match=name + words):
            torch.func.jvp(f, (x,), (torch.ones_like(x),))


def test_forward_mode_is_refused():
    _refuses_tangents("cpu")


@pytest.mark.gpu
def test_forward_mode_is_refused_on_the_gpu(hip_lib):
    print("case: tangents, also of a cotangent", flush=True)
    _refuses_tangents("cuda")
    x = torch.randn(3, 8, device="cuda", requires_grad=True)
    i = torch.zeros(3, dtype=torch.int64, device="cuda")
    t = torch.zeros(3, 4, device="cuda")
    for name, out in (("layer_norm", layer_norm(x)),
                      ("token_logprobs", token_logprobs(x, i).entropy),
                      ("distill_loss", distill_loss(x, t.long(), t).loss)):
        with torch.autograd.forward_ad.dual_level():
            cot = torch.autograd.forward_ad.make_dual(
                torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(TypeError, match=name):
                torch.autograd.grad(out, x, cot)


def test_temperatures_outside_the_range_are_refused(lib):
    P = 4096  # nothing is read before every check has passed
    for temp in (0.0, 9e-31, 1.1e30, float("inf"), float("nan")):
        for rc in (
                lib.rwkv7m_token_logprobs(1, 1, 3, 50, 0, 50, P, P, 2, temp,
                                          P, P, P, P, None, None),
                lib.rwkv7m_token_logprobs_backward(
                    1, 1, 3, 50, 0, 50, P, P, temp, P, P, P, P, P, None),
                lib.rwkv7m_distill_loss(1, 0, 1, 3, 50, 0, 50, 4, P, P, P,
                                        None, temp, P, P, P, None),
                lib.rwkv7m_distill_loss_backward(
                    1, 0, 1, 3, 50, 0, 50, 4, P, P, P, None, temp, P, 0, P,
                    None)):
            _refused(lib, rc, 1, "temperature must be within 1e-30 and 1e30")

"""HIP (gfx950) kernels around a language model's head: ctypes binding of the
``rwkv7m_layer_norm*``, ``rwkv7m_token_logprobs*`` and
``rwkv7m_distill_loss*`` entry points of librwkv7m_wkv.so
(include/rwkv7m_lm_head.h).

``x`` and ``logits`` are read where they lie as long as their last axis is
dense and their leading axes are one or two strided axes of rows (a
contiguous tensor, a slice of its columns, ``logits[:, :-1]``); other layouts
are copied first.  Every other tensor is made contiguous.  Tensors are torch
device tensors; there is no CPU fallback.
"""

from __future__ import annotations

import torch

from . import wkv_hip

MAX_TOP_K = 64
MAX_TEACHER_K = 256

_CODES = {torch.float32: wkv_hip.DTYPE_F32, torch.bfloat16:
          wkv_hip.DTYPE_BF16}


def _code(what: str, t: torch.Tensor) -> int:
    code = _CODES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what} must be bfloat16 or float32, got {t.dtype}")
    return code


def _call(dev, fn: str, *args) -> None:
    lib = wkv_hip.load_library()
    with wkv_hip._on(dev):
        rc = getattr(lib, fn)(*args, wkv_hip._stream(dev))
    wkv_hip._check(rc, fn)


def _rows(t: torch.Tensor):
    """(tensor, outer, inner, outer_stride, inner_stride) of the rows along
    the last axis; the tensor is ``t``, or a contiguous copy where its rows
    do not lie along two axes."""
    n = t.shape[-1]
    if not t.is_contiguous():
        axes = []  # (size, stride) from the innermost, adjoining ones merged
        for size, stride in zip(reversed(t.shape[:-1]),
                                reversed(t.stride()[:-1])):
            if size == 1:
                continue
            if axes and stride == axes[-1][0] * axes[-1][1]:
                axes[-1] = (axes[-1][0] * size, axes[-1][1])
            else:
                axes.append((size, stride))
        if len(axes) <= 2 and (n == 1 or t.stride(-1) == 1):
            (inner, istride), (outer, ostride) = (axes + [(1, 0)] * 2)[:2]
            return t, outer, inner, ostride, istride
        t = t.contiguous()
    return t, 1, t.numel() // n, 0, n


def _row_width(what: str, t: torch.Tensor) -> int:
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f"{what} must have at least one element along its "
                         f"last axis, got shape {tuple(t.shape)}")
    return t.shape[-1]


def _norm_params(x, weight, bias):
    """The parameters' dtype code; both of one dtype and C elements."""
    C, code = x.shape[-1], None
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.shape != (C,):
            raise ValueError(f"{name} must have shape {(C,)}, got "
                             f"{tuple(p.shape)}")
        if code is not None and p.dtype != weight.dtype:
            raise TypeError(f"weight and bias must share one dtype, got "
                            f"{weight.dtype} and {p.dtype}")
        code = _code(name, p)
    return wkv_hip.DTYPE_F32 if code is None else code


def layer_norm_forward(x, weight, bias, eps: float, with_stats: bool):
    """(y like x, mean, rstd): the statistics fp32 ``[rows]``, or None."""
    C = _row_width("x", x)
    code, pcode = _code("x", x), _norm_params(x, weight, bias)
    dev = wkv_hip._dev([t for t in (x, weight, bias) if t is not None])
    x, *rows = _rows(x)
    weight, bias = (None if p is None else p.contiguous()
                    for p in (weight, bias))
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    mean = rstd = None
    if with_stats:
        stats = torch.empty(2, rows[0] * rows[1], dtype=torch.float32,
                            device=dev)
        mean, rstd = stats.unbind()
    P = wkv_hip._p
    _call(dev, "rwkv7m_layer_norm", code, pcode, rows[0], rows[1], C, rows[2],
          rows[3], P(x), P(weight), P(bias), float(eps), P(y), P(mean),
          P(rstd))
    return y, mean, rstd


def layer_norm_backward(x, weight, bias_dtype, mean, rstd, dy,
                        want=(True, True, True)):
    """(dx like x, dweight ``[C]``, dbias ``[C]``), None where not wanted.
    ``bias_dtype`` is the bias's dtype, or None without one."""
    C = _row_width("x", x)
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError(f"dy has shape {tuple(dy.shape)} and dtype "
                         f"{dy.dtype}; expected {tuple(x.shape)} {x.dtype}")
    pdtype = bias_dtype if weight is None else weight.dtype
    code, pcode = _code("x", x), _norm_params(x, weight, None)
    if weight is None and bias_dtype is not None:
        pcode = _CODES[bias_dtype]
    dev = wkv_hip._dev([t for t in (x, weight, mean, rstd, dy)
                        if t is not None])
    x, *rows = _rows(x)
    n = rows[0] * rows[1]
    if mean.numel() != n or rstd.numel() != n:
        raise ValueError(f"mean and rstd must have {n} elements")
    dy = dy.contiguous()
    weight = None if weight is None else weight.contiguous()
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if want[0] else None
    dw, db = (torch.empty(C, dtype=pdtype, device=dev) if w else None
              for w in want[1:])
    ws, floats = None, 0
    if want[1] or want[2]:
        floats = wkv_hip.load_library().rwkv7m_layer_norm_workspace_floats(
            n, C)
        ws = torch.empty(max(floats, 1), dtype=torch.float32, device=dev)
    P = wkv_hip._p
    _call(dev, "rwkv7m_layer_norm_backward", code, pcode, rows[0], rows[1], C,
          rows[2], rows[3], P(x), P(weight), P(mean), P(rstd), P(dy), P(dx),
          P(dw), P(db), P(ws), floats)
    return dx, dw, db


def _ids(what: str, t: torch.Tensor, shape) -> torch.Tensor:
    """int64 contiguous ids of ``shape``."""
    if t.shape != shape:
        raise ValueError(f"{what} must have shape {tuple(shape)}, got "
                         f"{tuple(t.shape)}")
    if t.dtype != torch.int64:
        if t.dtype != torch.int32:
            raise TypeError(f"{what} must be int64 or int32, got {t.dtype}")
        t = t.long()
    return t.contiguous()


def _f32(what: str, t, shape):
    if t is None:
        return None
    if t.shape != shape:
        raise ValueError(f"{what} must have shape {tuple(shape)}, got "
                         f"{tuple(t.shape)}")
    return t.detach().to(torch.float32).contiguous()


def token_logprobs_forward(logits, tokens, top_k: int, temperature: float,
                           with_stats: bool):
    """(logprobs, entropy, top_ids, top_logprobs, stats): fp32 and int64
    ``[...]`` and ``[..., top_k]`` (None with top_k 0), and the backward's
    statistics or None."""
    V = _row_width("logits", logits)
    code, shape = _code("logits", logits), logits.shape[:-1]
    tokens = _ids("tokens", tokens, shape)
    dev = wkv_hip._dev([logits, tokens])
    logits, *rows = _rows(logits)

    def f32(*s):
        return torch.empty(s, dtype=torch.float32, device=dev)

    lp, ent = f32(*shape), f32(*shape)
    ids = top = stats = None
    if top_k:
        if top_k < 0 or top_k > min(V, MAX_TOP_K):
            raise ValueError(f"top_k must be within 0 and {min(V, MAX_TOP_K)}"
                             f" (V={V}), got {top_k}")
        ids = torch.empty(*shape, top_k, dtype=torch.int64, device=dev)
        top = f32(*shape, top_k)
    if with_stats:
        stats = f32(rows[0] * rows[1], 2)
    P = wkv_hip._p
    _call(dev, "rwkv7m_token_logprobs", code, rows[0], rows[1], V, rows[2],
          rows[3], P(logits), P(tokens), top_k, float(temperature), P(lp),
          P(ent), P(ids), P(top), P(stats))
    return lp, ent, ids, top, stats


def token_logprobs_backward(logits, tokens, temperature: float, stats,
                            entropy, d_logprobs, d_entropy):
    """dlogits like logits; either cotangent may be None."""
    V = _row_width("logits", logits)
    code, shape = _code("logits", logits), logits.shape[:-1]
    tokens = _ids("tokens", tokens, shape)
    dlp = _f32("d_logprobs", d_logprobs, shape)
    dent = _f32("d_entropy", d_entropy, shape)
    entropy = _f32("entropy", entropy, shape)
    dev = wkv_hip._dev([t for t in (logits, tokens, stats, entropy, dlp, dent)
                        if t is not None])
    logits, *rows = _rows(logits)
    if stats.shape != (rows[0] * rows[1], 2):
        raise ValueError("stats must be those of token_logprobs_forward")
    d = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
    P = wkv_hip._p
    _call(dev, "rwkv7m_token_logprobs_backward", code, rows[0], rows[1], V,
          rows[2], rows[3], P(logits), P(tokens), float(temperature),
          P(stats), P(entropy), P(dlp), P(dent), P(d))
    return d


def _distill_inputs(logits, ids, teacher, weight):
    V = _row_width("logits", logits)
    code, shape = _code("logits", logits), logits.shape[:-1]
    if teacher.dim() != logits.dim() or teacher.shape[:-1] != shape:
        raise ValueError(f"teacher_logits must have shape {tuple(shape)} "
                         f"with K alternatives behind, got "
                         f"{tuple(teacher.shape)}")
    K = teacher.shape[-1]
    if K > MAX_TEACHER_K:
        raise ValueError(f"at most {MAX_TEACHER_K} teacher alternatives are "
                         f"supported, got {K}")
    tcode = _code("teacher_logits", teacher)
    ids = _ids("teacher_ids", ids, teacher.shape)
    teacher = teacher.contiguous()
    weight = _f32("weight", weight, shape)
    dev = wkv_hip._dev([t for t in (logits, ids, teacher, weight)
                        if t is not None])
    logits, *rows = _rows(logits)
    P = wkv_hip._p
    args = (code, tcode, rows[0], rows[1], V, rows[2], rows[3], K, P(logits),
            P(ids), P(teacher), P(weight))
    return dev, shape, args, (logits, ids, teacher, weight)


def distill_loss_forward(logits, teacher_ids, teacher_logits, weight,
                         temperature: float, with_grad: bool):
    """(loss fp32 scalar, row_losses fp32 [...], dlogits or None)."""
    dev, shape, args, keep = _distill_inputs(logits, teacher_ids,
                                             teacher_logits, weight)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    rows = torch.empty(shape, dtype=torch.float32, device=dev)
    d = torch.empty(logits.shape, dtype=logits.dtype, device=dev) \
        if with_grad else None
    P = wkv_hip._p
    _call(dev, "rwkv7m_distill_loss", *args, float(temperature), P(loss),
          P(rows), P(d))
    return loss, rows, d


def distill_loss_backward(logits, teacher_ids, teacher_logits, weight,
                          temperature: float, scale, dlogits=None):
    """The gradient of scale * loss; ``dlogits``, if given, already holds
    the loss's own and is what is returned."""
    dev, _, args, keep = _distill_inputs(logits, teacher_ids, teacher_logits,
                                         weight)
    scale = _f32("scale", scale, ())
    wkv_hip._dev([logits, scale])
    held = dlogits is not None
    if held and (dlogits.shape != logits.shape or
                 dlogits.dtype != logits.dtype or
                 not dlogits.is_contiguous() or dlogits.device != dev):
        raise ValueError("dlogits must be distill_loss_forward's")
    if not held:
        dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
    P = wkv_hip._p
    _call(dev, "rwkv7m_distill_loss_backward", *args, float(temperature),
          P(scale), int(held), P(dlogits))
    return dlogits

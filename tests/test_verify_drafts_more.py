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

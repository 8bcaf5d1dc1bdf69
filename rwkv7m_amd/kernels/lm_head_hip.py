"""HIP (gfx950) kernels around a language model's head: the torch binding of
the ``rwkv7m_layer_norm*``, ``rwkv7m_token_logprobs*`` and
``rwkv7m_distill_loss*`` entry points of librwkv7m_wkv.so
(include/rwkv7m_lm_head.h), built from csrc/torch_lm_head.cpp.

``load_binding()`` returns the compiled module; its functions check their
arguments, allocate their outputs, launch on the current stream and record
their autograd nodes.  Activations and logits are read where they lie as long
as their last axis is dense and their leading axes are one or two strided
axes of rows (a contiguous tensor, a slice of its columns, ``logits[:,
:-1]``); other layouts are copied first.  There is no CPU fallback.
"""

from __future__ import annotations

import importlib.util
import os

from . import wkv_hip

_PKG_DIR = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BINDING_PATH = os.path.join(_PKG_DIR, "_lm_head_torch.so")

_binding = None


def load_binding():
    """The binding's module.  Raises ``RuntimeError`` if it is not built."""
    global _binding
    if _binding is None:
        wkv_hip.load_library()
        if not os.path.exists(BINDING_PATH):
            raise RuntimeError(
                f"torch binding not found at {BINDING_PATH}; build it with "
                "`python -m rwkv7m_amd._build` (or __graft_entry__.build())")
        spec = importlib.util.spec_from_file_location("_lm_head_torch",
                                                      BINDING_PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        _binding = module
    return _binding

"""The gated delta rule's scale and memory at their limits (without a GPU; no
valid request is made)."""

from __future__ import annotations

import ctypes

import pytest

from test_gated_delta_refusals import P, _inputs, _refused, lib  # noqa: F401


@pytest.mark.parametrize("scale", [3.5e38, -1e39, 1e300])
def test_a_scale_past_fp32_is_refused(lib, scale):  # noqa: F811
    """The kernels hold it in fp32: it would be an infinity there."""
    x = ctypes.byref(_inputs(scale=scale))
    stride = (ctypes.c_int64 * 3)(640, 128, 32)
    for rc in (lib.rwkv7m_gated_delta_rule(x, None, None, None, None, None, 0,
                                           None),
               lib.rwkv7m_gated_delta_rule_backward(
                   x, None, stride, None, None, None, None, None, None, None,
                   None, None, 0, None),
               lib.rwkv7m_gated_delta_step(x, 2, None, None, None, 1, None,
                                           None)):
        _refused(lib, rc, 1, "scale is not finite")


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("Hk,Hv,Dk,Dv,T", [(2, 2, 64, 64, 64), (1, 3, 72, 40, 65),
                                           (4, 4, 128, 256, 1000)])
def test_memory_as_documented(lib, dtype, Hk, Hv, Dk, Dv, T):  # noqa: F811
    """38144 bytes of matrices a value head and chunk; for a backward 4 Dv (Dk +
    64) more, Dk and Dv rounded up, which it takes again, and 8 Hv Dk a token
    where value heads share key heads."""
    B = 2
    x = ctypes.byref(_inputs(dtype=dtype, B=B, T=T, Hk=Hk, Hv=Hv, Dk=Dk,
                             Dv=Dv))
    chunks = B * Hv * -(-T // 64)
    dk, dv = (64 if Dk <= 64 else 128), -(-Dv // 32) * 32
    kept = chunks * 4 * dv * (dk + 64)
    assert lib.rwkv7m_gated_delta_workspace_bytes(x, 0) == 38144 * chunks
    assert 4 * lib.rwkv7m_gated_delta_saved_floats(x) == kept + 38144 * chunks
    shared = 8 * B * T * Hv * Dk if Hv > Hk else 0
    assert lib.rwkv7m_gated_delta_workspace_bytes(x, 1) == kept + shared

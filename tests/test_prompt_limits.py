"""Limits of the entry points around a prompt at their borders, without a GPU."""
import ctypes as C

import pytest

from tests.test_prompt_args import EINVAL, EWORKSPACE, P, Q


def prompt_desc(N, **kw):
    return N.PromptAttentionDesc(**{**dict(dtype=16, seqs=1, heads=8, kv_heads=2, head_dim=64, causal=1, q_rows=16, kv_rows=4000, scale=0.125,
                                           q_stride=512, k_stride=128, v_stride=128, o_stride=512), **kw})


@pytest.mark.parametrize("scale,taken", [(2.0 ** 127, True), (-2.0 ** 127, True), (2.0 ** 127 * 1.01, False), (-3.4e38, False), (float("inf"), False),
                                         (float("nan"), False), (0.0, True)])
def test_scales(native, scale, taken):
    """scale log2 e has to be a number of fp32. The call asks for a workspace and gets none, so that it ends before a launch."""
    d = prompt_desc(native, scale=scale)
    L = native.lib()
    assert (L.spinn_hip_prompt_attention_workspace_size(C.byref(d)) > 0) == taken
    rc = L.spinn_hip_prompt_attention(C.byref(d), P, P, P, P, P, Q, None, None, 0, None)
    assert rc == (EWORKSPACE if taken else EINVAL)

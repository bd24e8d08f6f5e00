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


def test_rows_of_a_launch(native):
    """One row more than spinn_hip_quantize_rows takes."""
    L = native.lib()
    for k, most in ((1, (1 << 26) - 4), (1024, (1 << 26) - 4), (1025, (1 << 24) - 1), (4096, (1 << 24) - 1), (4097, (1 << 22) - 1)):
        ldq = (k + 15) // 16 * 16
        assert L.spinn_hip_quantize_rows(1, most + 1, k, P, k, Q, ldq, P, None) == -2, (k, most)


@pytest.mark.parametrize("change,taken", [({}, True), (dict(seqs=1 << 24), True), (dict(seqs=(1 << 24) + 1), False), (dict(kv_rows=1 << 30), True),
                                          (dict(kv_rows=(1 << 30) + 1), False), (dict(q_stride=1 << 24), True), (dict(q_stride=(1 << 24) + 1), False),
                                          (dict(q_stride=511), False), (dict(seqs=0, q_rows=1 << 27), True), (dict(seqs=0, q_rows=(1 << 27) + 1), False)], ids=str)
def test_prompt_sizes(native, change, taken):
    """A call without rows or sequences ends well where its descriptor is taken."""
    d = prompt_desc(native, **{"q_rows": 0, **change})
    assert native.lib().spinn_hip_prompt_attention(C.byref(d), P, P, P, P, P, Q, None, None, 0, None) == (0 if taken else EINVAL)

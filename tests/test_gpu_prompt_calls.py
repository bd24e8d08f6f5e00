"""Calls around a prompt that the header allows and that lie off the usual ones: no keys at all, heads before tokens, another stream than the first."""
import ctypes as C

import pytest
import torch

from tests.decodeops import BF16, F16, F32, NAMES, assert_close, gen, ptr, randn, stream
from tests.promptops import Prompt, quantize_ref, rope_frequencies, rope_ref
from tests.test_gpu_linear_i8 import ints, layer, quantize
from tests.test_gpu_rope import desc, run, table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("dim", [64, 128, 33])
def test_no_keys_at_all(hip, dtype, dim):
    """kv_rows = 0 and no arrays of keys and values: zeros, and a logarithm of nothing."""
    p = Prompt(gen(1), dtype, [5, 200], 4, 2, dim, lead=2, tail=1)
    starts = torch.tensor(p.starts, dtype=torch.int32, device="cuda")
    none = torch.zeros_like(starts)
    d = hip.PromptAttentionDesc(dtype=dtype, seqs=2, heads=4, kv_heads=2, head_dim=dim, causal=1, q_rows=p.rows, kv_rows=0, scale=1.0,
                                q_stride=p.q.stride(0), k_stride=2 * dim, v_stride=2 * dim, o_stride=p.o.stride(0))
    assert hip.lib().spinn_hip_prompt_attention_workspace_size(C.byref(d)) == 0
    hip.check(hip.lib().spinn_hip_prompt_attention(C.byref(d), ptr(p.q), None, None, ptr(starts), ptr(none), ptr(p.o), ptr(p.lse), None, 0, stream()), "prompt")
    assert (p.o[2:-1] == 0).all() and (p.o[:2] == 7).all() and (p.o[-1] == 7).all()
    assert (p.lse[2:-1] == -float("inf")).all() and (p.lse[:2] == 7).all()


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("inter", [0, 1], ids=["half", "interleaved"])
def test_rope_heads_before_tokens(hip, inter, in_place):
    """[heads, tokens, dim]: a head's tokens next to each other."""
    heads, tokens, dim, rot = 5, 37, 48, 32
    x = randn(gen(2), heads, tokens, dim, dtype=BF16).cuda()
    before = x.cpu().transpose(0, 1)
    y = x if in_place else torch.zeros_like(x)
    position = torch.arange(tokens, dtype=torch.int32, device="cuda") * 3
    d = desc(hip, BF16, heads, dim, rot, inter, strides=(dim, tokens * dim, dim, tokens * dim))
    run(hip, d, position, table(hip, d), x, y)
    want, tol = rope_ref(before, position.cpu(), rope_frequencies(rot, 10000.0, 0, 1.0, 1.0, 4.0, 512), rot, inter, 1.0, BF16)
    got = y.cpu().transpose(0, 1)
    assert torch.equal(got[..., rot:], before[..., rot:])
    assert_close(got[..., :rot], want[..., :rot], tol[..., :rot], "heads before tokens")


def test_layers_on_two_streams(hip):
    """Quantisation and a layer with a workspace of its own on two streams, several times over."""
    g = gen(3)
    m, n, k = 200, 1024, 8192
    jobs = []
    for _ in range(2):
        x, w = randn(g, m, k, dtype=BF16).cuda(), ints(g, n, k).cuda()
        jobs.append((x, w, torch.rand(n, generator=g).cuda(), torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        got = []
        for x, w, sw, s in jobs:
            with torch.cuda.stream(s):
                q, sx = quantize(hip, x)
                got.append(layer(hip, q, sx, w, sw, F32, k=k))
    torch.cuda.synchronize()
    for (x, w, sw, _), y in zip(jobs, got):
        q, sx = quantize_ref(x.cpu())
        v = (q.cuda().double() @ w.double().t().contiguous()) * sx.cuda().double()[:, None] * sw.double()
        assert_close(y, v, 4 * 2.0 ** -24 * v.abs() + 1e-37, "two streams")

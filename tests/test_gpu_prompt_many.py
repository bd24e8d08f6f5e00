"""spinn_hip_prompt_attention over very many short sequences, and what their search may cost."""
import ctypes as C

import pytest
import torch

from tests.decodeops import BF16, HALF_STEP, ptr, stream

pytestmark = pytest.mark.gpu

HEADS, DIM = 2, 32


def call(N, starts, q, k, v, o):
    d = N.PromptAttentionDesc(dtype=BF16, seqs=starts.numel() - 1, heads=HEADS, kv_heads=1, head_dim=DIM, causal=1, q_rows=q.shape[0],
                              kv_rows=q.shape[0], scale=0.3, q_stride=HEADS * DIM, k_stride=DIM, v_stride=DIM, o_stride=HEADS * DIM)
    assert N.lib().spinn_hip_prompt_attention_workspace_size(C.byref(d)) == 0
    N.check(N.lib().spinn_hip_prompt_attention(C.byref(d), ptr(q), ptr(k), ptr(v), ptr(starts), None, ptr(o), None, None, 0, stream()), "prompt")


def packed(seqs, most, lead=3, tail=2):
    """Sequences of 0 to `most` rows."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seqs)
    lens = torch.randint(0, most + 1, (seqs,), generator=g, device="cuda")
    starts = torch.cat([lens.new_zeros(1), lens.cumsum(0)]) + lead
    rows = int(starts[-1]) + tail
    q, k, v = (torch.randn(rows, w, generator=g, device="cuda").bfloat16() for w in (HEADS * DIM, DIM, DIM))
    return lens, starts.to(torch.int32), q, k, v, torch.full_like(q, 7.0)


@pytest.mark.parametrize("seqs", [65, 4095, 4096, 4097, 100000, 262145])
def test_sequences_of_up_to_two_rows(hip, seqs):
    """A first row gives its value as it is, a second one the mean of two under sigmoid(difference): the weights' rounding and the
    result's, half a step each, and 2^-18 of the values for fp32's."""
    lens, starts, q, k, v, o = packed(seqs, 2)
    call(hip, starts, q, k, v, o)
    first = starts[:-1].long()
    one = first[lens > 0]
    assert torch.equal(o[one].view(-1, HEADS, DIM), v[one][:, None].expand(-1, HEADS, DIM))
    two = first[lens == 2]
    a, b = two, two + 1
    q2 = q[b].double().view(-1, HEADS, DIM)
    p = torch.sigmoid(0.3 * (q2 * (k[b] - k[a].double())[:, None]).sum(-1, keepdim=True))
    va, vb = v[a].double()[:, None], v[b].double()[:, None]
    want, size = (1 - p) * va + p * vb, (1 - p) * va.abs() + p * vb.abs()
    tol = HALF_STEP[BF16] * (size + want.abs() * (1 + HALF_STEP[BF16])) + 2.0 ** -18 * size
    assert ((o[b].view(-1, HEADS, DIM).double() - want).abs() <= tol).all()
    inside = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
    inside[3:-2] = True
    assert (o[~inside] == 7).all()


def test_a_million_sequences(hip):
    """A workgroup's search among them is a few steps: all of them are done in a fraction of a second."""
    seqs = 1 << 20
    starts = torch.arange(seqs + 1, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    q, k, v = (torch.randn(seqs, w, generator=g, device="cuda").bfloat16() for w in (HEADS * DIM, DIM, DIM))
    o = torch.zeros_like(q)
    call(hip, starts[:101], q[:100], k[:100], v[:100], o[:100])  # the kernel is loaded
    torch.cuda.synchronize()
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    call(hip, starts, q, k, v, o)
    end.record()
    torch.cuda.synchronize()
    assert torch.equal(o.view(seqs, HEADS, DIM), v[:, None].expand(-1, HEADS, DIM))
    assert begin.elapsed_time(end) < 500

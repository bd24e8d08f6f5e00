"""The operators around a prompt where rows lie past 2^32 bytes, and where many short sequences meet many keys."""
import random

import pytest
import torch

from tests.decodeops import BF16, F32, assert_close, gen, ptr, randn, stream
from tests.promptops import Prompt, quantize_ref, rope_frequencies, rope_ref
from tests.test_gpu_kv_assign import State, call, compare
from tests.test_gpu_linear_i8 import ints, layer
from tests.test_gpu_prompt import check
from tests.test_gpu_rope import desc, run, table

pytestmark = pytest.mark.gpu


def apart(body, stride):
    """The rows of `body`, `stride` elements apart."""
    out = torch.empty((body.shape[0] - 1) * stride + body.shape[1], dtype=body.dtype, device="cuda").as_strided(body.shape, (stride, 1))
    out.copy_(body)
    return out


@pytest.mark.parametrize("dtype,stride,far", [(BF16, 1 << 22, "kv"), (F32, 1 << 22, "kv"), (BF16, 1 << 24, "qo"), (BF16, (1 << 23) + 8, "qo"), (F32, (1 << 22) + 1, "kvqo")])
def test_attention_rows_far_apart(hip, dtype, stride, far):
    """Keys, values, queries and results whose last rows lie past 2^32 bytes."""
    p = Prompt(gen(3), dtype, [170, 1, 129], 2, 1, 64, lead=2, tail=1, kv_lens=[250, 260, 70] if "kv" in far else None)
    if "kv" in far:
        p.k, p.v = apart(p.k, stride), apart(p.v, stride)
    if "qo" in far:
        p.q, p.o = apart(p.q, stride), apart(p.o, stride)
    check(hip, p, 0.125, 1, what=f"rows {stride} apart")


def short_over_many(seqs, keys):
    """Some without rows, some of few keys."""
    lens = [(i * 7) % 3 for i in range(seqs)]
    kv_lens = [keys + 10 * (i % 50) if i % 9 else 5 for i in range(seqs)]
    return Prompt(gen(seqs), BF16, lens, 2, 1, 64, kv_lens=kv_lens, tail=2)


@pytest.mark.parametrize("seqs", [65, 70, 120])
def test_many_short_sequences(hip, seqs):
    """More sequences than lanes, more keys than rows."""
    check(hip, short_over_many(seqs, 1400), 0.125, 1, what=f"{seqs} sequences")


@pytest.mark.parametrize("seqs", [65, 70, 120])
def test_many_short_sequences_over_many_keys(hip, seqs):
    """The same with keys that are split and joined."""
    p = short_over_many(seqs, 2600)
    check(hip, p, 0.125, 1, what=f"{seqs} sequences over many keys")
    assert p.ws is not None, "not split"


def test_starts_that_do_not_ascend(hip):
    """Outside the contract, but such a call ends, and the next one is right."""
    g = gen(1)
    for seqs in (40, 3000):
        p = Prompt(g, BF16, [1] * seqs, 2, 1, 32, tail=3)
        p.run(hip, 0.2, 1, starts=torch.randint(-10, 4000, (seqs + 1,), generator=g, dtype=torch.int32).tolist())
        p.run(hip, 0.2, 1, starts=[0, seqs + 3] * (seqs // 2) + [0])
        p.o.fill_(7.0)
        p.lse.fill_(7.0)
        check(hip, p, 0.2, 1, what="after such a call")


def test_rope_rows_far_apart(hip):
    tokens, heads, dim, stride = 70, 3, 64, (1 << 25) + 8
    x = apart(randn(gen(2), tokens, heads * dim, dtype=BF16).cuda(), stride)
    position = torch.arange(tokens, dtype=torch.int32, device="cuda") * 1000
    before = x.cpu().reshape(tokens, heads, dim)
    d = desc(hip, BF16, heads, dim, dim, 0, strides=(stride, dim, stride, dim))
    run(hip, d, position, table(hip, d), x, x)
    want, tol = rope_ref(before, position.cpu(), rope_frequencies(dim, 10000.0, 0, 1.0, 1.0, 4.0, 512), dim, 0, 1.0, BF16)
    assert_close(x.cpu().reshape(want.shape), want, tol, "rope far apart")


@pytest.mark.parametrize("m", [40, 260])
def test_linear_rows_far_apart(hip, m):
    """Rows of 8-bit integers and of results past 2^32 bytes, quantised there."""
    stride = 1 << (28 if m == 40 else 25)
    n, k = 70, 200
    g = gen(m)
    values = randn(g, m, k, dtype=F32)
    xq = apart(torch.zeros(m, 208, dtype=torch.int8), stride)
    scale = torch.zeros(m, device="cuda")
    hip.check(hip.lib().spinn_hip_quantize_rows(F32, m, k, ptr(values.cuda()), k, ptr(xq), stride, ptr(scale), stream()), "quantize")
    want_q, want_s = quantize_ref(values)
    assert torch.equal(xq[:, :k].cpu(), want_q) and torch.equal(scale.cpu(), want_s)
    w, one = ints(g, n, k), torch.ones(n, device="cuda")
    y = apart(torch.zeros(m, n), 1 << 23 if m > 100 else 1 << 26)
    layer(hip, xq, torch.ones(m, device="cuda"), w.cuda(), one, F32, k=k, y=y)
    assert torch.equal(y.cpu(), (want_q.double() @ w.double().t()).float())


def test_pages_for_the_most_sequences(hip):
    """65536 sequences at once, a page each, and all of them ended."""
    st = State(random.Random(3), 65536, 4, 1, 60000, lengths=[0] * 65536)
    dev = st.device()
    for new in ([1] * 65536, [-1] * 65536):
        want = st.step(new, 65536)
        compare(st, dev, call(hip, st, dev, new, 65536), want, 65536)

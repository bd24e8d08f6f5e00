"""spinn_hip_prompt_attention on the GPU against 64 bits; the bounds are derived in promptops.prompt_ref."""
import math

import pytest
import torch

from tests.decodeops import BF16, F16, F32, NAMES, assert_close, gen
from tests.promptops import Prompt

pytestmark = pytest.mark.gpu


def check(N, p, scale, causal, lse=True, what=""):
    p.run(N, scale, causal, lse)
    o, o_tol, lse_ref, lse_tol = p.ref(scale, causal)
    inside = torch.zeros(p.rows, dtype=torch.bool)
    inside[p.starts[0]:p.starts[-1]] = True
    got = p.o.cpu().reshape(p.rows, p.heads, p.dim)
    assert_close(got[inside], o[inside], o_tol[inside], f"o {NAMES[p.dtype]} {what}")
    assert (got[~inside] == 7).all(), "rows outside the sequences were written"
    if lse:
        some = inside[:, None] & (lse_ref != -math.inf)
        assert_close(p.lse.cpu()[some], lse_ref[some], lse_tol[some], f"lse {what}")
        assert (p.lse.cpu()[inside[:, None] & (lse_ref == -math.inf)] == -math.inf).all()
        assert (p.lse.cpu()[~inside] == 7).all()
    else:
        assert (p.lse == 7).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("causal", [1, 0], ids=["causal", "full"])
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 64), (4, 1, 128), (6, 2, 80), (8, 8, 32), (3, 1, 96), (5, 1, 256), (2, 2, 160), (16, 1, 64), (40, 1, 16)])
def test_heads(hip, dtype, causal, heads, kv, dim):
    """Head groups and sizes over ragged lengths, among them one token and none."""
    p = Prompt(gen(heads * dim), dtype, [70, 1, 0, 33, 129, 2], heads, kv, dim, lead=3, tail=5)
    check(hip, p, 2 * dim ** -0.5, causal, what=f"{heads}/{kv}x{dim}")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 400])
def test_lengths(hip, dtype, n):
    """Lengths around every tile's border, whole and causal."""
    for causal in (0, 1):
        check(hip, Prompt(gen(n), dtype, [n], 2, 1, 64), 0.25, causal, what=f"n {n}")


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
def test_long(hip, dtype):
    """A longer sequence, whose maximum moves many times: keys that grow along the sequence, and shrink."""
    for sign in (1.0, -1.0):
        p = Prompt(gen(5), dtype, [1500], 2, 1, 64)
        grow = torch.linspace(0.1, 3.0, 1500, device="cuda")[:, None]
        p.k.copy_((p.k.float() * (grow if sign > 0 else grow.flip(0))).to(p.k.dtype))
        check(hip, p, 0.5, 1, what="growing")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
@pytest.mark.parametrize("causal", [1, 0], ids=["causal", "full"])
def test_other_key_lengths(hip, dtype, causal):
    """Keys of their own lengths: more than rows (a prompt that goes on), fewer (rows that see none), none at all."""
    p = Prompt(gen(6), dtype, [10, 100, 7, 64, 3, 0], 4, 2, 64, kv_lens=[300, 40, 0, 64, 1, 9], lead=2, tail=4)
    check(hip, p, 0.3, causal, what="kv lengths")


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("dim,pad,offset,fused", [(64, 0, 0, True), (64, 8, 0, True), (64, 5, 0, False), (128, 0, 1, True), (33, 0, 0, True), (80, 3, 3, False),
                                                  (3, 0, 0, False), (1, 1, 0, False), (7, 0, 1, True), (130, 0, 0, True), (255, 1, 0, False)])
def test_strides_and_alignment(hip, dtype, dim, pad, offset, fused):
    """Rows of a fused projection, wider buffers, any alignment, heads that are no whole 16-byte runs."""
    p = Prompt(gen(dim), dtype, [50, 90], 4, 2, dim, pad=pad, offset=offset, fused=fused, lead=1, tail=1)
    before = p.o.as_strided((p.rows, p.o.stride(0)), (p.o.stride(0), 1)) if not offset else None
    check(hip, p, dim ** -0.5, 1, what=f"dim {dim} pad {pad} offset {offset}")
    if before is not None and pad:
        assert (before[:-1, 4 * dim:] == 7).all()  # between the rows of o


@pytest.mark.parametrize("seqs", [63, 64, 65, 200, 5000])
def test_many_sequences(hip, seqs):
    """More sequences than lanes, empty ones among them."""
    g = gen(seqs)
    lens = torch.randint(0, 5 if seqs > 1000 else 40, (seqs,), generator=g).tolist()
    lens[seqs // 2] = 150
    p = Prompt(g, BF16, lens, 2, 1, 32, tail=3)
    check(hip, p, 0.2, 1, what=f"{seqs} sequences")


def test_all_empty(hip):
    p = Prompt(gen(1), BF16, [0, 0, 0], 2, 1, 32, lead=4, tail=2)
    p.run(hip, 1.0, 1)
    assert (p.o == 7).all() and (p.lse == 7).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30, 3.0])
def test_scales(hip, dtype, scale):
    """No scale (all weights equal), a negative one, the least, a large one."""
    for causal in (0, 1):
        check(hip, Prompt(gen(2), dtype, [40, 150], 2, 2, 48), scale, causal, what=f"scale {scale}")


@pytest.mark.parametrize("dtype", [F16, BF16], ids=NAMES.get)
def test_equal_weights(hip, dtype):
    """One value everywhere: the weights add up to one, so the result is the value, rounded once."""
    p = Prompt(gen(3), dtype, [777], 1, 1, 64)
    p.v.fill_(1.7)
    p.run(hip, 1e-3, 1)
    want = float(p.v[0, 0])
    step = {F16: 2.0 ** -10, BF16: 2.0 ** -7}[dtype]
    assert ((p.o.float() - want).abs() <= step * want).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
def test_large_scores(hip, dtype):
    """Scores in the thousands: one key takes all; and such that differ by little on a large level."""
    p = Prompt(gen(4), dtype, [100, 60], 2, 1, 64)
    check(hip, p, 30.0, 1, what="large")
    p.k.copy_((p.k.float() * 0.01 + 20.0).to(p.k.dtype))
    p.q.copy_(p.q.abs())
    check(hip, p, 0.25, 1, what="level")


def test_many_small_weights_fp16(hip):
    """A sink that takes most, thousands of keys of tiny weight whose sum counts."""
    p = Prompt(gen(7), F16, [4000], 1, 1, 64)
    p.q.fill_(1.0)
    p.k.zero_()
    p.k[0].fill_(0.175)  # 11.2 above all others
    p.v.fill_(1.0)
    p.v[0].fill_(0.0)
    check(hip, p, 1.0, 0, what="small weights")


def test_rows_outside_are_not_read(hip):
    """Infinities and NaN before, behind and between: only a sequence's own rows count."""
    for bad in (math.nan, math.inf):
        p = Prompt(gen(8), BF16, [33, 65, 20], 4, 2, 64, lead=40, tail=70)
        check(hip, p, 0.2, 1, what="surrounded")
        # the middle sequence's keys and values are broken: the others are as they were
        want = p.o.clone()
        a, b = p.starts[1], p.starts[2]
        p.k[a:b] = bad
        p.v[a:b] = bad
        p.o.fill_(7.0)
        p.run(hip, 0.2, 1)
        assert torch.equal(p.o[:a], want[:a]) and torch.equal(p.o[b:], want[b:])


def test_starts_out_of_range(hip):
    """Starts are cut to the rows that there are; what they name beyond is neither read nor written."""
    p = Prompt(gen(9), BF16, [30, 40, 50], 2, 1, 64, lead=0, tail=0)
    p.run(hip, 0.2, 1, starts=[-5, 30, 70, 100000])
    got = p.o.clone()
    p.o.fill_(7.0)
    p.run(hip, 0.2, 1)
    assert torch.equal(got, p.o)
    p.o.fill_(7.0)
    p.run(hip, 0.2, 1, starts=[500, 600, 700, 800])
    assert (p.o == 7).all()


def test_repeats(hip):
    """The same call gives the same bits."""
    p = Prompt(gen(10), BF16, [200, 900, 31], 8, 2, 128)
    p.run(hip, 0.2, 1)
    first = p.o.clone()
    for _ in range(5):
        p.o.fill_(0)
        p.run(hip, 0.2, 1)
        assert torch.equal(first, p.o)


def test_streams_at_once(hip):
    """Two calls on two streams, each with its own workspace."""
    ps = [Prompt(gen(20 + i), BF16, [300 + 50 * i, 77], 8, 2, 64) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ps]
    for _ in range(3):
        for p, s in zip(ps, streams):
            with torch.cuda.stream(s):
                p.run(hip, 0.3, 1)
    torch.cuda.synchronize()
    for p in ps:
        o, tol, _, _ = p.ref(0.3, 1)
        assert_close(p.o.cpu().reshape(o.shape), o, tol, "streams")


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("causal", [1, 0], ids=["causal", "full"])
@pytest.mark.parametrize("lens,kv_lens,heads,kv,dim", [([3], [5000], 4, 2, 64), ([1], [2500], 1, 1, 128), ([1, 0, 20, 7], [3000, 100, 9000, 0], 8, 2, 80),
                                                       ([130], [4100], 2, 1, 96), ([5, 5], [1300, 3000], 3, 3, 33), ([2], [2600], 2, 1, 256)], ids=str)
def test_few_rows_over_many_keys(hip, dtype, causal, lens, kv_lens, heads, kv, dim):
    """Keys split over workgroups and joined: parts of ordinary length, short and empty ones, sequences without keys."""
    p = Prompt(gen(len(lens) + dim), dtype, lens, heads, kv, dim, kv_lens=kv_lens, lead=1, tail=2)
    check(hip, p, dim ** -0.5, causal, what=f"few rows {lens} {kv_lens}")
    assert p.ws is not None, "not split"
    first, lse = p.o.clone(), p.lse.clone()
    p.run(hip, dim ** -0.5, causal)
    assert torch.equal(first, p.o) and torch.equal(lse.view(torch.int32), p.lse.view(torch.int32))


def test_captured_with_other_lengths(hip):
    """A captured call replayed while the starts in memory change; its workspace dirtied between the replays."""
    import ctypes as C

    from tests.decodeops import ptr, stream, workspace
    p = Prompt(gen(11), BF16, [40, 40], 4, 2, 64, kv_lens=[2000, 3000])
    for rows in ((p.rows, p.kv_rows), (p.rows, p.kv_rows // 16)):  # split and not
        d = hip.PromptAttentionDesc(dtype=BF16, seqs=2, heads=4, kv_heads=2, head_dim=64, causal=1, q_rows=rows[0], kv_rows=rows[1], scale=0.2,
                                    q_stride=p.q.stride(0), k_stride=p.k.stride(0), v_stride=p.v.stride(0), o_stride=p.o.stride(0))
        size = hip.lib().spinn_hip_prompt_attention_workspace_size(C.byref(d))
        ws = workspace(size)
        starts, kv_starts = (torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(2))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            hip.check(hip.lib().spinn_hip_prompt_attention(C.byref(d), ptr(p.q), ptr(p.k), ptr(p.v), ptr(starts), ptr(kv_starts), ptr(p.o), None,
                                                           ptr(ws), size, stream()), "prompt")
        for a, b in (([0, 40, 80], [0, rows[1] // 3, rows[1]]), ([0, 1, 30], [0, 70, 90]), ([5, 5, 80], [0, 0, rows[1]])):
            starts.copy_(torch.tensor(a, dtype=torch.int32))
            kv_starts.copy_(torch.tensor(b, dtype=torch.int32))
            p.o.fill_(7.0)
            if ws is not None:
                ws.fill_(0xFF)
            graph.replay()
            torch.cuda.synchronize()
            p.starts, p.kv_starts = a, b
            o, tol, _, _ = p.ref(0.2, 1)
            got = p.o.cpu().reshape(o.shape)
            assert_close(got[a[0]:a[2]], o[a[0]:a[2]], tol[a[0]:a[2]], f"replay {a} {b}")
            assert (got[a[2]:] == 7).all() and (got[:a[0]] == 7).all()

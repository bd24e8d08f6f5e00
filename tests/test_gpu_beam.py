"""spinn_hip_beam_select and spinn_hip_beam_reorder against a stable sort of 64-bit keys.

Scores: a key's sum of exponentials is off by at most 2^-20 of itself (the exponentials' arguments and values in
fp32, added in 64 bits), and the result is rounded to fp32: 2^-20 + 2^-23 |key|."""
import ctypes as C
import math

import pytest
import torch

from tests.decodeops import BF16, F16, F32, NAMES, TORCH, beam_ref, gen, ptr, stream, workspace

pytestmark = pytest.mark.gpu


def select(N, dtype, logits, scores, k, finished=None, end=0, stride=None):
    """One call and its comparison."""
    L = N.lib()
    b, w, v = logits.shape
    stride = stride or v
    x = torch.full((b * w, stride), 1e4, device="cuda").to(TORCH[dtype])
    x[:, :v] = logits.reshape(b * w, v).cuda()
    d = N.BeamDesc(dtype=dtype, batch=b, beams=w, vocab=v, k=k, end_token=end, logits_stride=stride)
    size = L.spinn_hip_beam_select_workspace_size(C.byref(d))
    ws = workspace(size)
    sd, fd = scores.cuda(), None if finished is None else finished.cuda()
    os = torch.full((b, k), 777.0, device="cuda")
    op, ot = (torch.full((b, k), 777, dtype=torch.int32, device="cuda") for _ in range(2))
    print(f"[beam] {NAMES[dtype]} {b}x{w}x{v} k={k} ws={size}", flush=True)
    N.check(L.spinn_hip_beam_select(C.byref(d), ptr(x), ptr(sd), ptr(fd), ptr(os), ptr(op), ptr(ot), ptr(ws), size, stream()),
            "spinn_hip_beam_select")
    torch.cuda.synchronize()
    key, parents, tokens = beam_ref(logits, scores, finished, end, k)
    assert torch.equal(op.cpu(), parents), (op.cpu(), parents, key)
    assert torch.equal(ot.cpu(), tokens), (ot.cpu(), tokens, key)
    got = os.cpu().double()
    assert torch.equal(got == -math.inf, key == -math.inf)
    off = torch.where(key == -math.inf, 0.0, (got - key).abs() - 2.0 ** -20 - 2.0 ** -23 * key.abs())
    assert (off <= 0).all(), off.max()


def make(seed, dtype, b, w, v, spread=2.5):
    g = gen(seed)
    return (torch.randn(b, w, v, generator=g) * spread).to(TORCH[dtype]), -10 * torch.rand(b, w, generator=g)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("b,w,v,k", [(1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 7, 20), (1, 4, 1000, 8), (3, 5, 32000, 10), (2, 8, 50001, 16),
                                     (1, 64, 2100, 128), (2, 2, 4096, 1), (40, 16, 513, 32)])
def test_select_sizes(hip, torch_gpu, dtype, b, w, v, k):
    select(hip, dtype, *make(v + k, dtype, b, w, v), k)


@pytest.mark.parametrize("b,w,v,k", [(8, 16, 40001, 128), (1, 64, 200001, 20), (8, 16, 40000, 24), (8, 16, 40000, 25)])
def test_select_long_lists(hip, torch_gpu, b, w, v, k):
    """The longest candidate lists on chip, more lists than the joining workgroup has lanes, and both sides of the
    chunk length that goes by k."""
    select(hip, F16, *make(v + k, F16, b, w, v), k)


@pytest.mark.parametrize("v,k", [(300001, 20), (200001, 128)])
@pytest.mark.parametrize("kind", ["ordinary", "equal", "few beams"])
def test_select_more_lists_than_lanes(hip, torch_gpu, v, k, kind):
    """64 beams of 19 and 25 chunks: more lists than the 1024 lanes of the joining workgroup, so that lanes have several."""
    x, s = make(v + k, F16, 1, 64, v)
    fin = torch.zeros(1, 64, dtype=torch.uint8)
    if kind == "equal":
        x = (torch.randint(0, 2, (1, 1, v), generator=gen(k)) * 0.5).half().expand(1, 64, v).contiguous()
        s[:] = -torch.arange(64).div(16, rounding_mode="floor")
    elif kind == "few beams":
        s[0, torch.arange(64) % 5 > 0] = -math.inf
        fin[0, ::10] = 1
    select(hip, F16, x, s, k, finished=fin, end=v - 2)


def test_select_many_chunks(hip, torch_gpu):
    """Rows cut into chunks of every length: by the rows' number, few or many workgroups."""
    for b in (1, 16, 64):
        select(hip, BF16, *make(b, BF16, b, 8, 40000), 16)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
def test_select_strides(hip, torch_gpu, dtype):
    for stride in (1000, 1003, 1008):
        select(hip, dtype, *make(stride, dtype, 2, 3, 999), 6, stride=stride)


@pytest.mark.parametrize("k", [1, 8, 16, 128])
def test_select_equal_keys(hip, torch_gpu, k):
    """Equal logits, equal beams: the lower beam, then the lower token."""
    flat = torch.zeros(1, 4, 9000)
    select(hip, F32, flat, torch.zeros(1, 4), k)
    g = gen(k)
    few = torch.randint(0, 3, (2, 4, 9000), generator=g).float()
    few[:, 1] = few[:, 0]
    few[:, 3] = few[:, 2]
    select(hip, F32, few, torch.tensor([[-1.0, -1.0, -2.0, -2.0]] * 2), k)
    zeros = torch.where(torch.rand(1, 2, 500, generator=g) < 0.5, 0.0, -0.0)
    select(hip, F32, zeros, torch.zeros(1, 2), k)


@pytest.mark.parametrize("k", [3, 64])
def test_select_one_thread_holds_the_best(hip, torch_gpu, k):
    """The best tokens side by side, and all in one beam."""
    x, s = make(k, F32, 1, 4, 30000)
    x[0, 2, 4096:4096 + 64] = 30 + torch.arange(64.0)
    select(hip, F32, x, s, k)
    for runs in (1, 8, 256):  # ascending rows, and rows that ascend within every run: parts of a chunk far above others
        y = torch.sort(x[0].reshape(4, 30000 // 8 // 25, -1), 2)[0].reshape(1, 4, 30000)
        y = y + (torch.arange(30000) // runs % 64).float() * 0.5
        select(hip, F32, y, s, k)
    x, s = make(k + 1, F32, 1, 4, 30000)
    x[0] = torch.sort(x[0], 1)[0]
    select(hip, F32, x, s, k)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
def test_select_masked_vocabularies(hip, torch_gpu, dtype):
    """Tokens hidden by -inf, all but a few or all of them, NaN, the type's least number, empty beams (the first step)."""
    x, s = make(3, dtype, 4, 4, 5000)
    x[0, :, 3:] = -math.inf
    x[1, 1] = -math.inf
    x[1, 2, ::2] = math.nan
    x[2, :, 10:] = torch.finfo(TORCH[dtype]).min
    x[3] = -math.inf
    s[0, 1:] = -math.inf
    s[2, 0] = math.nan
    select(hip, dtype, x, s, 8)
    select(hip, dtype, x[:, :1].contiguous(), torch.zeros(4, 1), 8)
    select(hip, dtype, x, torch.full((4, 4), -math.inf), 8)


def test_select_huge_logits(hip, torch_gpu):
    """+inf counts as the largest finite number; spreads at which all but the best exponential vanish."""
    x, s = make(4, F32, 2, 3, 4000, spread=1e4)
    select(hip, F32, x, s, 6)
    x[0, 1, 77] = math.inf
    select(hip, F32, x[:1], s[:1], 1)


def far_ref(logits, scores, k):
    """beam_ref without finished beams, the logits' maximum taken off before the sum's logarithm: a key of 64 bits, at any
    magnitude."""
    x = logits.double()
    key = scores.double()[:, :, None] + torch.log_softmax(x, 2)
    val, at = torch.sort(key.flatten(1), dim=1, descending=True, stable=True)
    return val[:, :k], (at[:, :k] // x.shape[2]).int(), (at[:, :k] % x.shape[2]).int()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
@pytest.mark.parametrize("far", [9e5, 1e6, 1.1e6, 1e9, 4e9, 5e9, 1e10, 1e12, 1e15, 1e20, 9e29, 2e30, 3e38])
@pytest.mark.parametrize("sign", [-1, 1])
def test_select_far_logits(hip, torch_gpu, dtype, far, sign):
    """Finite logits far from the others, as programs hide tokens with: single ones, whole chunks, whole rows, beside an
    ordinary beam."""
    for b, v in ((1, 40000), (64, 20000)):  # chunks of 2048 tokens, and of the longest
        x, s = make(int(far % 997) + v, dtype, b, 4, v)
        hidden = torch.tensor(sign * far).to(TORCH[dtype])
        x[:, 0, 100:110] = hidden
        x[:, 1, 4096:20000] = hidden  # chunks between others (from 16384 on of the longest), and the row's end there
        x[:, 2] = hidden
        x[:, 2, 5] = hidden * (1 + sign * 2.0 ** -6)  # next to it
        s[:] = torch.tensor([-1.0, -3.0, -5.0, -7.0])
        k = 24
        L, xd, sd = hip.lib(), x.cuda(), s.cuda()
        d = hip.BeamDesc(dtype=dtype, batch=b, beams=4, vocab=v, k=k, end_token=0, logits_stride=v)
        size = L.spinn_hip_beam_select_workspace_size(C.byref(d))
        ws, os = workspace(size), torch.full((b, k), 777.0, device="cuda")
        op, ot = (torch.full((b, k), 777, dtype=torch.int32, device="cuda") for _ in range(2))
        hip.check(L.spinn_hip_beam_select(C.byref(d), ptr(xd), ptr(sd), None, ptr(os), ptr(op), ptr(ot), ptr(ws), size, stream()),
                  "spinn_hip_beam_select")
        key, parents, tokens = far_ref(x, s, k)
        got = os.cpu().double()
        assert torch.isfinite(got).all()
        # as in select(): the sum of exponentials, and the result's rounding
        assert ((got - key).abs() <= 2.0 ** -20 + 2.0 ** -23 * key.abs()).all(), (got - key).abs().max()
        assert torch.equal(op.cpu(), parents) and torch.equal(ot.cpu(), tokens)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("v", [8, 40, 999, 8000, 40000])
def test_select_signalling_nans(hip, torch_gpu, dtype, v):
    """NaN of every kind count as -inf: among ordinary logits, and in rows of a single other logit, which an ordinary
    maximum with a signalling NaN loses."""
    x, s = make(v, dtype, 2, 4, v)
    bits = torch.int32 if dtype == F32 else torch.int16
    quiet = {F32: 0x7fc00000, F16: 0x7e00, BF16: 0x7fc0}[dtype]
    for i, nan in enumerate((quiet, quiet ^ (quiet & -quiet) | 1, -1, quiet - 1)):  # quiet, signalling, negative, signalling
        lone = x[0, i].clone()
        lone[:] = -math.inf
        lone[v // 3] = -2.5
        x[0, i] = lone
        x[0, i].view(bits)[torch.arange(v) % 3 != (v // 3) % 3] = nan
        x[1, i].view(bits)[torch.arange(v) % 5 < 2] = nan
    assert x[0].isnan().any(1).all() and x[1].isnan().any(1).all()
    select(hip, dtype, x, s, 8)


@pytest.mark.parametrize("end", [0, 999])
def test_select_finished(hip, torch_gpu, end):
    """Ended beams go on with the end token alone; all ended; ended and empty."""
    x, s = make(5, F16, 4, 4, 1000)
    fin = torch.zeros(4, 4, dtype=torch.uint8)
    fin[0, 1], fin[1, :], fin[2, 0], fin[2, 3] = 1, 255, 1, 1
    s[2, 3] = -math.inf
    s[0, 1] = 0.0
    select(hip, F16, x, s, 8, finished=fin, end=end)


def test_select_join_list_overflows(hip, torch_gpu):
    """More candidates above the bound than the joining workgroup lists: few of its threads hold all the best."""
    # 64 beams of one chunk each; one beam far above the others
    x, s = make(6, F32, 1, 64, 2000)
    s[0] = -1000 - 20 * torch.arange(64.0)
    select(hip, F32, x, s, 128)
    s[0, 40:] = torch.randn(24)
    select(hip, F32, x, s, 128)


# ---- reordering ----

@pytest.mark.parametrize("row", [1, 3, 4, 16, 100, 4096, 70000, 2000001])
def test_reorder(hip, torch_gpu, row):
    """Bytes of rows inside wider ones; parents outside the beams leave their rows as they were."""
    N, L, g = hip, hip.lib(), gen(row)
    b, w, k = 3, 4, 6
    src = torch.randint(0, 256, (b * w, row + 5), generator=g, dtype=torch.uint8)
    tab = torch.randint(0, 1000, (b * w, 7), generator=g, dtype=torch.int32)
    parents = torch.randint(0, w, (b, k), generator=g, dtype=torch.int32)
    parents[0, 0], parents[1, 2], parents[2, 5] = -1, w, 2 ** 31 - 1
    sd, td, pd = src.cuda(), tab.cuda(), parents.cuda()
    dst = torch.full((b * k, row + 16), 7, dtype=torch.uint8, device="cuda")
    dtab = torch.full((b * k, 7), 7, dtype=torch.int32, device="cuda")
    states = (N.BeamState * 3)(N.BeamState(ptr(sd), ptr(dst), row, row + 5, row + 16), N.BeamState(None, None, 0, 0, 0),
                               N.BeamState(ptr(td), ptr(dtab), 28, 28, 28))
    N.check(L.spinn_hip_beam_reorder(states, 3, b, w, k, ptr(pd), stream()), "reorder")
    torch.cuda.synchronize()
    want, wtab = torch.full((b * k, row + 16), 7, dtype=torch.uint8), torch.full((b * k, 7), 7, dtype=torch.int32)
    for i in range(b):
        for j in range(k):
            p = int(parents[i, j])
            if 0 <= p < w:
                want[i * k + j, :row] = src[i * w + p, :row]
                wtab[i * k + j] = tab[i * w + p]
    assert torch.equal(dst.cpu(), want) and torch.equal(dtab.cpu(), wtab)


@pytest.mark.parametrize("states,batch,k", [(1, 1 << 20, 4), (5, 1 << 20, 4), (16, 1 << 18, 9)])
def test_reorder_most_rows(hip, torch_gpu, states, batch, k):
    """Up to 2^22 rows of up to 16 states, more shares than a launch has workgroups of 256 threads."""
    N, L, w = hip, hip.lib(), 4
    g = torch.Generator(device="cuda")
    g.manual_seed(states)
    parents = torch.randint(0, w, (batch, k), generator=g, device="cuda", dtype=torch.int32)
    parents[::7, 1] = -1
    src = [torch.randint(0, 1 << 30, (batch, w), generator=g, device="cuda", dtype=torch.int32) for _ in range(states)]
    dst = [torch.full((batch, k), -5, device="cuda", dtype=torch.int32) for _ in range(states)]
    table = (N.BeamState * states)(*[N.BeamState(ptr(s), ptr(d), 4, 4, 4) for s, d in zip(src, dst)])
    N.check(L.spinn_hip_beam_reorder(table, states, batch, w, k, ptr(parents), stream()), "reorder")
    for s, d in zip(src, dst):
        assert torch.equal(d, torch.where(parents >= 0, s.gather(1, parents.clamp(min=0).long()), -5))

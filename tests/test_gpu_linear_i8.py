"""spinn_hip_quantize_rows and spinn_hip_linear_i8 on the GPU against 64 bits."""
import ctypes as C
import math

import pytest
import torch

from tests.decodeops import ACTS, BF16, F16, F32, HALF_STEP, NAMES, TORCH, assert_close, gen, ptr, randn, stream, workspace
from tests.promptops import quantize_ref

pytestmark = pytest.mark.gpu


def quantize(N, x, pad=0):
    rows, k = x.shape
    ldq = (k + 15) // 16 * 16 + pad
    q = torch.full((rows, ldq), 99, dtype=torch.int8, device="cuda")
    s = torch.full((rows,), 7.0, device="cuda")
    code = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}[x.dtype]
    N.check(N.lib().spinn_hip_quantize_rows(code, rows, k, ptr(x), x.stride(0), ptr(q), ldq, ptr(s), stream()), "quantize")
    assert (q[:, (k + 15) // 16 * 16:] == 99).all()  # nothing behind the padded row
    return q, s


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("rows,k,pad,offset", [(1, 1, 0, 0), (3, 7, 0, 0), (5, 16, 0, 1), (64, 64, 8, 0), (7, 1000, 1, 0), (9, 1024, 0, 0), (6, 1025, 3, 5),
                                               (3, 4096, 0, 0), (2, 4099, 0, 1), (5, 16384, 0, 0), (2, 16400, 0, 0), (2, 70001, 1, 1)])
def test_quantize(hip, dtype, rows, k, pad, offset):
    """Whole numbers and scales equal the definition's, rows of any length and alignment."""
    flat = randn(gen(rows * k), offset + rows * (k + pad), dtype=dtype).cuda()
    x = flat[offset:].view(rows, k + pad)[:, :k]
    q, s = quantize(hip, x, 16)
    want, scale = quantize_ref(x.cpu())
    assert torch.equal(s.cpu(), scale)
    assert torch.equal(q[:, :k].cpu(), want)
    assert (q[:, k:(k + 15) // 16 * 16] == 0).all()


def test_quantize_borders(hip):
    """Quotients at and next to halves: ties to even of the exact quotient, whatever its fp32 rounding says."""
    for scale in (1.0, 0.75, 3.1415927e-3, 1.7e20, 2.0 ** -90):
        s = torch.tensor(scale, dtype=torch.float32)
        top = (s.double() * 127).float()
        s = (top.double() / 127).float()
        half = (torch.arange(-126, 127).double() + 0.5) * s.double()
        row = [top.view(1)]
        for v in (half.float(), torch.nextafter(half.float(), torch.tensor(math.inf)), torch.nextafter(half.float(), torch.tensor(-math.inf))):
            row.append(v)
        x = torch.cat(row)[None].cuda()
        q, got = quantize(hip, x)
        want, ws = quantize_ref(x.cpu())
        assert torch.equal(got.cpu(), ws) and torch.equal(q[:, :x.shape[1]].cpu(), want), scale


def test_quantize_special_rows(hip):
    """Rows of zeros, of the least numbers, of the largest, with an infinity or a NaN."""
    tiny = torch.finfo(torch.float32).tiny
    rows = [[0.0, -0.0, 0.0, 0.0], [2.0 ** -149, -2.0 ** -149, 0.0, 2.0 ** -148], [127 * 2.0 ** -149, 63.0 * 2.0 ** -149, 2.0 ** -149, 0.0],
            [200 * 2.0 ** -149, 100 * 2.0 ** -149, -3 * 2.0 ** -149, 0.0], [tiny, -tiny / 2, tiny / 3, tiny / 254], [1e-31, 3e-32, -5e-33, 1e-35],
            [3.4e38, -3.4e38, 1e38, 1.3e36], [1.0, math.inf, 2.0, 3.0], [1.0, 2.0, math.nan, 3.0], [-math.inf, math.nan, 0.0, 0.0], [1.0, 2.0, 3.0, 4.0]]
    x = torch.tensor(rows).repeat(1, 5)
    q, s = quantize(hip, x.cuda())
    want, scale = quantize_ref(x)
    assert torch.equal(s.cpu().isnan(), scale.isnan()) and torch.equal(s.cpu().nan_to_num(9), scale.nan_to_num(9))
    assert torch.equal(q[:, :20].cpu(), want)


# ---- layers ----

def pack(N, d, w):
    L = N.lib()
    size = L.spinn_hip_linear_i8_packed_size(C.byref(d))
    packed = torch.full((size,), 0xA5, device="cuda", dtype=torch.uint8)
    N.check(L.spinn_hip_linear_i8_pack_weights(C.byref(d), ptr(w), ptr(packed), stream()), "pack")
    return packed


def layer(N, x, sx, w, sw, dtype, trans_w=1, act=0, bias=None, res=None, y=None, ldx=None, k=None, packed=None, ws_fill=0xA5):
    m, k = x.shape[0], k or x.shape[1]
    n = sw.numel()
    y = torch.full((m, n), 7.0, dtype=TORCH[dtype], device="cuda") if y is None else y
    d = N.LinearI8Desc(m=m, n=n, k=k, dtype=dtype, trans_w=trans_w, act=act, ldx=x.stride(0), ldres=res.stride(0) if res is not None else 0,
                       ldy=y.stride(0) if m > 1 else 0)
    packed = pack(N, d, w) if packed is None else packed
    L = N.lib()
    size = L.spinn_hip_linear_i8_workspace_size(C.byref(d))
    ws = workspace(size, ws_fill)
    N.check(L.spinn_hip_linear_i8(C.byref(d), ptr(x), ptr(sx), ptr(packed), ptr(sw), ptr(bias), ptr(res), ptr(y), ptr(ws), size, stream()), "linear_i8")
    return y


def ints(g, *shape):
    return torch.randint(-128, 128, shape, generator=g, dtype=torch.int8)


def padded(x, poison=77):
    """Rows of whole 16-byte runs, what is behind k arbitrary."""
    m, k = x.shape
    out = torch.full((m, (k + 15) // 16 * 16), poison, dtype=torch.int8, device="cuda")
    out[:, :k] = x.cuda()
    return out


SHAPES = [(1, 1, 1), (1, 64, 128), (2, 65, 130), (16, 100, 64), (17, 257, 1000), (33, 2048, 512), (64, 96, 4096), (65, 512, 2048), (130, 129, 65),
          (200, 1024, 16384), (300, 700, 300), (512, 4096, 256), (1000, 4100, 128), (257, 8192, 384), (2100, 8200, 192)]


@pytest.mark.parametrize("m,n,k", SHAPES, ids=str)
@pytest.mark.parametrize("trans_w", [1, 0])
def test_exact_sums(hip, m, n, k, trans_w):
    """Scales of one: sums of 32 bits, rounded to fp32 once. What lies behind k in a row of x does not count."""
    g = gen(m + n + k)
    x, w = ints(g, m, k), ints(g, n, k)
    one = torch.ones(max(m, n), device="cuda")
    y = layer(hip, padded(x), one[:m], (w if trans_w else w.t().contiguous()).cuda(), one[:n], F32, trans_w, k=k)
    want = (x.cuda().double() @ w.cuda().double().t().contiguous()).float()
    assert torch.equal(y, want)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("m,n,k", [(1, 200, 96), (40, 333, 500), (200, 1024, 4096), (700, 1030, 260)], ids=str)
def test_epilogue(hip, dtype, act, m, n, k):
    """Scales, bias, residual and activation. The bound: the sum's conversion, two scales, bias and residual are five roundings of 2^-24 of the
    magnitudes' sum; the activation's slope of at most 1.13 and 2^-19 of its argument; the result's rounding."""
    g = gen(m + n + k + act)
    x, w = ints(g, m, k), ints(g, n, k)
    sx, sw = torch.rand(m, generator=g) + 0.5, (torch.rand(n, generator=g) + 0.5) / (5000 * k ** 0.5)
    bias, res = randn(g, n, dtype=dtype), randn(g, m, n, dtype=dtype)
    y = layer(hip, padded(x), sx.cuda(), w.cuda(), sw.cuda(), dtype, 1, act, bias.cuda(), res.cuda(), k=k)
    v = (x.double() @ w.double().t()) * sx.double()[:, None] * sw.double()
    s = v.abs() + bias.double().abs() + res.double().abs()
    v = v + bias.double() + res.double()
    off = 5 * 2.0 ** -24 * s * 1.13 + 2.0 ** -19 * v.abs() * (act not in (0, 1))
    ref = ACTS[act](v)
    assert_close(y, ref, off + HALF_STEP[dtype] * (ref.abs() + off) + 2.0 ** -25 * (dtype == F16) + 1e-37, f"linear_i8 {m}x{n}x{k} act {act}")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
def test_strides_and_places(hip, dtype):
    """Rows of x, residual and y in wider buffers of odd strides; y over its residual; nothing else written."""
    g = gen(9)
    for m, n, k in ((5, 70, 48), (150, 300, 200)):
        wide = torch.full((m, (k + 15) // 16 * 16 + 32), 55, dtype=torch.int8, device="cuda")
        x, w = ints(g, m, k), ints(g, n, k)
        wide[:, :k] = x.cuda()
        sx, sw = torch.rand(m, generator=g).cuda(), torch.rand(n, generator=g).cuda() / k
        buf = randn(g, m, n + 3, dtype=dtype).cuda()
        before = buf.clone()
        y = buf[:, 1:n + 1]
        plain = layer(hip, wide[:, :k], sx, w.cuda(), sw, dtype, res=before[:, 1:n + 1].contiguous(), k=k)
        layer(hip, wide[:, :k], sx, w.cuda(), sw, dtype, res=y, y=y, k=k)
        assert torch.equal(y, plain)
        assert torch.equal(buf[:, 0], before[:, 0]) and torch.equal(buf[:, n + 1:], before[:, n + 1:])


def test_special_scales(hip):
    """A scale of NaN makes its row or column NaN and no other; of zero leaves bias alone."""
    g = gen(10)
    for m, n, k in ((3, 40, 64), (140, 300, 256)):
        x, w = ints(g, m, k), ints(g, n, k)
        sx, sw = torch.ones(m), torch.ones(n)
        sx[1], sx[2], sw[5] = math.nan, 0.0, 0.0
        bias = randn(g, n)
        y = layer(hip, padded(x), sx.cuda(), w.cuda(), sw.cuda(), F32, bias=bias.cuda(), k=k).cpu()
        assert y[1].isnan().all() and y[[0] + list(range(2, m))].isfinite().all()
        assert torch.equal(y[2], bias) and torch.equal(y[0, 5], bias[5])


def test_largest_k(hip):
    """Sums of the largest products over the longest rows stay within 32 bits."""
    k = hip.I8_MAX_K
    one = torch.ones(64, device="cuda")
    for m in (1, 40):
        x = torch.full((m, k + 1), -128, dtype=torch.int8, device="cuda")
        w = torch.full((8, k), -128, dtype=torch.int8, device="cuda")
        y = layer(hip, x, one[:m], w, one[:8], F32, k=k)
        assert (y.double() == float(torch.tensor(16384.0 * k).float())).all()


def test_quantized_layer_end_to_end(hip):
    """x and w quantised on the device: the result is that of the numbers they stand for, within the roundings of the epilogue; the
    quantisation itself is off by at most half a step of each row, which bounds the distance from the unquantised layer."""
    g = gen(11)
    m, n, k = 37, 300, 520
    x, w = randn(g, m, k, dtype=BF16), randn(g, n, k, dtype=BF16)
    xq, sx = quantize(hip, x.cuda())
    wq, sw = quantize(hip, w.cuda())
    wk = wq[:, :k].contiguous()
    y = layer(hip, xq, sx, wk, sw, F32, k=k).cpu().double()
    xs, ws = xq[:, :k].cpu().double() * sx.cpu().double()[:, None], wk.cpu().double() * sw.cpu().double()[:, None]
    ref = xs @ ws.t()
    assert_close(y, ref, 3 * 2.0 ** -24 * ref.abs() + 1e-37, "quantised layer")
    hx, hw = sx.cpu().double()[:, None] / 2 * (1 + 1e-6), sw.cpu().double()[:, None] / 2 * (1 + 1e-6)
    far = hx * ws.abs().sum(1) + (xs.abs().sum(1)[:, None] + k * hx) * hw.t()
    assert ((y - x.double() @ w.double().t()).abs() <= far + 1e-6).all()


def test_captured_and_replayed(hip):
    """Quantisation and a layer that splits K, captured; the workspace dirtied between the replays."""
    g = gen(12)
    m, n, k = 200, 1024, 16384
    d = hip.LinearI8Desc(m=m, n=n, k=k, dtype=BF16, trans_w=1)
    L = hip.lib()
    w = ints(g, n, k).cuda()
    packed = pack(hip, d, w)
    size = L.spinn_hip_linear_i8_workspace_size(C.byref(d))
    assert size > 0
    ws = workspace(size)
    x = torch.zeros((m, k), dtype=torch.bfloat16, device="cuda")
    xq, sx = torch.empty((m, k), dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")
    sw = torch.rand(n, generator=g).cuda()
    y = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")

    def step(to):
        hip.check(L.spinn_hip_quantize_rows(BF16, m, k, ptr(x), k, ptr(xq), k, ptr(sx), stream()), "quantize")
        hip.check(L.spinn_hip_linear_i8(C.byref(d), ptr(xq), ptr(sx), ptr(packed), ptr(sw), None, None, ptr(to), ptr(ws), size, stream()), "layer")

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(y)
    for seed in range(3):
        x.copy_(randn(gen(seed), m, k, dtype=BF16))
        ws.fill_(0xFF)
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.empty_like(y)
        step(eager)
        assert torch.equal(y, eager)

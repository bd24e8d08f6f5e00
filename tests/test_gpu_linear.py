"""spinn_hip_linear against the formula in 64 bits: types, layouts, ragged sizes, strides, epilogues.

The bound of each element is derived in tests/decodeops.py (linear_ref)."""
import ctypes as C
import math

import pytest
import torch

from tests.decodeops import BF16, F16, F32, NAMES, TORCH, assert_close, gen, linear_pack, linear_ref, ptr, randn, stream, workspace

pytestmark = pytest.mark.gpu


def run(N, dtype, m, n, k, act=0, bias=False, res=False, trans_w=1, padx=0, padr=0, pady=0, off=0, seed=0, in_place=False):
    """One call on rows of wider buffers; everything around y has to stay as it was."""
    L, g, t = N.lib(), gen(seed + 7919 * m + 31 * n + k), TORCH[dtype]
    x = randn(g, m, k + padx, dtype=dtype)
    w = randn(g, *((n, k) if trans_w else (k, n)), dtype=dtype, scale=k ** -0.5)
    b = randn(g, n, dtype=dtype) if bias else None
    r = randn(g, m, n + padr, dtype=dtype) if res else None
    if in_place:
        pady = padr
    xb = torch.full((off + m * (k + padx),), float("nan"), dtype=t, device="cuda")
    xd = xb[off:].view(m, k + padx)
    xd.copy_(x)
    if padx:
        xd[:, k:] = float("nan")  # behind a row: not read into any sum
    rd = None if r is None else r.cuda()
    yd = rd if in_place else torch.full((m + 2, n + pady), 777.0, dtype=t, device="cuda")
    d = N.LinearDesc(m=m, n=n, k=k, dtype=dtype, trans_w=trans_w, act=act, x_unaligned=int(off % (16 // t.itemsize) != 0),
                     ldx=k + padx, ldres=n + padr, ldy=n + pady)
    packed = linear_pack(N, d, w.cuda())
    size = L.spinn_hip_linear_workspace_size(C.byref(d))
    ws = workspace(size)
    print(f"[linear] {NAMES[dtype]} m={m} n={n} k={k} act={act} ws={size}", flush=True)
    y0 = yd if in_place else yd[1:]
    N.check(L.spinn_hip_linear(C.byref(d), ptr(xd), ptr(packed), ptr(None if b is None else b.cuda()), ptr(rd), ptr(y0),
                               ptr(ws), size, stream()), "spinn_hip_linear")
    torch.cuda.synchronize()
    ref, tol = linear_ref(x[:, :k], w, trans_w, b, None if r is None else r[:, :n], act, dtype)
    assert_close(y0[:m, :n], ref, tol, f"{NAMES[dtype]} {m}x{n}x{k}")
    if in_place:
        assert torch.equal(yd[:, n:].cpu(), r[:, n:])
    else:
        assert (yd[0] == 777).all() and (yd[m + 1] == 777).all() and (yd[:, n:] == 777).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("mnk", [(1, 1, 1), (1, 1000, 2048), (3, 17, 31), (16, 64, 64), (17, 65, 96), (33, 130, 257),
                                 (64, 256, 128), (65, 300, 520), (128, 128, 64), (300, 200, 72), (1000, 1030, 200)], ids=str)
def test_linear_sizes(hip, torch_gpu, dtype, mnk):
    run(hip, dtype, *mnk, act=3, bias=True)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
@pytest.mark.parametrize("mnk", [(2048, 4096, 96), (4100, 4200, 64), (1030, 1100, 136)], ids=str)
def test_linear_many_tiles(hip, torch_gpu, dtype, mnk):
    """Grids on the large tiles, with rows, columns and K that end inside one."""
    run(hip, dtype, *mnk, bias=True, res=True)


@pytest.mark.parametrize("act", [0, 1, 3, 6, 7])
@pytest.mark.parametrize("bias,res", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("m", [5, 70, 600])
def test_linear_epilogue(hip, torch_gpu, act, bias, res, m):
    run(hip, F16, m, 520, 64, act=act, bias=bias, res=res)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("m", [4, 90, 700])
@pytest.mark.parametrize("trans_w", [0, 1])
def test_linear_weight_layouts(hip, torch_gpu, dtype, m, trans_w):
    run(hip, dtype, m, 333, 100, trans_w=trans_w, bias=True)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
@pytest.mark.parametrize("m", [2, 100, 520])
@pytest.mark.parametrize("padx,padr,pady,off", [(8, 0, 0, 0), (5, 0, 0, 0), (0, 3, 5, 0), (0, 8, 16, 0), (0, 0, 0, 3), (8, 4, 4, 8)])
def test_linear_strides(hip, torch_gpu, dtype, m, padx, padr, pady, off):
    """Rows inside wider buffers, x off its 16-byte boundary, residual and y in runs of 4 and not."""
    run(hip, dtype, m, 260, 128, res=True, bias=True, padx=padx, padr=padr, pady=pady, off=off)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("mnk", [(5, 70, 3), (40, 200, 7), (2, 50, 8), (1, 100, 16385), (16, 100, 4097), (9, 64, 1023), (33, 300, 2047),
                                 (60, 4200, 301), (427, 131, 275)], ids=str)
def test_linear_loose_rows(hip, torch_gpu, dtype, mnk):
    """Few rows that are no whole runs: read where they are, up to the length from which they are laid out first."""
    run(hip, dtype, *mnk, bias=True, padx=1, off=1)


@pytest.mark.parametrize("m", [1, 200, 600])
def test_linear_in_place(hip, torch_gpu, m):
    """y over its own residual, the residual stream of a network."""
    run(hip, BF16, m, 256, 192, res=True, bias=True, padr=8, in_place=True)


# Layers that run on tiles of the matrix cores on a device of 256 CUs, K long enough for the loop's steady part: (m, n, k),
# whether K is split (the sums then go through the workspace).
TILES = [((130, 260, 2056), True), ((200, 1024, 4104), True),  # 64 x 128, split
         ((70, 8200, 2056), False), ((1030, 1100, 4000), False), ((1568, 2048, 512), False),  # 64 x 128 whole, up to one per CU and more
         ((2048, 4096, 1000), False), ((1100, 4300, 776), False),  # 128 x 128
         ((4100, 4200, 520), False)]  # 256 x 256


def tiles_on(N, dtype, m, n, k, split, x_unaligned=0):
    """The workspace beside laid-out rows of x holds the parts of a split, 4 bytes of every element of its tiles each."""
    d = N.LinearDesc(m=m, n=n, k=k, dtype=dtype, trans_w=1, x_unaligned=x_unaligned)
    size = N.lib().spinn_hip_linear_workspace_size(C.byref(d))
    e = TORCH[dtype].itemsize
    laid = 0
    if x_unaligned or k * e % 16:
        laid = (m + 15) // 16 * 16 * -(-k * e // 128) * 128
    part = (m + 63) // 64 * 64 * (-(-n // 128) * 128) * 4
    assert size >= laid and (size - laid) % part == 0
    assert (size - laid) // part >= 2 if split else size == laid


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("mnk,split", TILES, ids=str)
def test_linear_tiles(hip, torch_gpu, dtype, mnk, split):
    """Rows of whole runs; rows, columns and K end inside tiles, K one run into a granule."""
    tiles_on(hip, dtype, *mnk, split)
    run(hip, dtype, *mnk, bias=True, res=True, act=1)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("mnk,split", TILES, ids=str)
def test_linear_tiles_loose_rows(hip, torch_gpu, dtype, mnk, split):
    """x laid out in the workspace first; K ends one element into a granule, or one before its end."""
    m, n, k = mnk
    for k in (k // 64 * 64 + 1, k // 64 * 64 - 1):
        tiles_on(hip, dtype, m, n, k, split, x_unaligned=1)
        run(hip, dtype, m, n, k, bias=True, padx=2, off=1, trans_w=k & 2 and 1)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
@pytest.mark.parametrize("mnk,split", [t for t in TILES if t[0][0] in (200, 1568, 1100, 4100)], ids=str)
@pytest.mark.parametrize("act,bias,res,in_place", [(0, False, False, False), (3, True, False, False), (6, False, True, True),
                                                   (7, True, True, True)])
def test_linear_tiles_epilogue(hip, torch_gpu, dtype, mnk, split, act, bias, res, in_place):
    tiles_on(hip, dtype, *mnk, split)
    run(hip, dtype, *mnk, act=act, bias=bias, res=res, padr=3 if in_place else 0, in_place=in_place)


@pytest.mark.parametrize("mnk,split", TILES, ids=str)
def test_linear_tiles_values(hip, torch_gpu, mnk, split):
    """Infinities and NaN on tiles reach the outputs of their row and column alone, at the ends of rows, columns and K, too."""
    N, L = hip, hip.lib()
    m, n, k = mnk
    g = gen(m)
    x, w = randn(g, m, k, dtype=BF16).cuda(), randn(g, n, k, dtype=BF16, scale=0.125).cuda()
    x[1, 5], x[m - 1, k - 1], x[m // 2, k // 2] = float("inf"), float("nan"), float("-inf")
    w[n - 1, k - 1], w[7, 9] = float("inf"), float("nan")
    d = N.LinearDesc(m=m, n=n, k=k, dtype=BF16, trans_w=1)
    packed = linear_pack(N, d, w)
    size = L.spinn_hip_linear_workspace_size(C.byref(d))
    ws, y = workspace(size, 0xFF), torch.full((m, n), 777.0, device="cuda", dtype=torch.bfloat16)
    N.check(L.spinn_hip_linear(C.byref(d), ptr(x), ptr(packed), None, None, ptr(y), ptr(ws), size, stream()), "linear")
    ref = torch.mm(x.float(), w.float().t().contiguous())
    assert torch.equal(y.isnan(), ref.isnan())
    assert torch.equal(torch.where(y.isinf(), y.float(), 0.0), torch.where(ref.isinf(), ref, 0.0))


def test_linear_far_rows(hip, torch_gpu):
    """Rows whose offsets pass 32 bits of bytes."""
    N, L = hip, hip.lib()
    m, n, k, ld = 3, 40, 64, 1 << 28
    buf = torch.zeros(2 * ld + 64, dtype=torch.float32, device="cuda")
    x = torch.as_strided(buf, (m, k), (ld, 1))
    g = gen(1)
    xc, w = randn(g, m, k), randn(g, n, k, scale=0.125)
    x.copy_(xc)
    d = N.LinearDesc(m=m, n=n, k=k, dtype=F32, trans_w=1, act=0, ldx=ld)
    packed = linear_pack(N, d, w.cuda())
    y = torch.empty(m, n, device="cuda")
    assert L.spinn_hip_linear_workspace_size(C.byref(d)) == 0
    N.check(L.spinn_hip_linear(C.byref(d), ptr(x), ptr(packed), None, None, ptr(y), None, 0, stream()), "linear")
    assert_close(y, *linear_ref(xc, w, 1, None, None, 0, F32), "far rows")


@pytest.mark.parametrize("act", [6, 7])
def test_linear_gelu_accuracy(hip, torch_gpu, act):
    """Both forms over a dense sweep, in fp32: the residual is the argument, x is zero.

    erf form: Phi near 0 is 1/2 + v S with v S <= 0.4 within 2.2 roundings (polynomial and fit), its sum and the product:
    under 3 * 2^-24 of |v|; further out Phi(-a) <= 0.11 within 10 roundings and the exponent's two of v^2 / 2: under
    (10 + v^2) 2^-24 of itself, so that 1 - Phi(-a) and the product stay under 3 * 2^-24 again.
    tanh form, v / (1 + e), e = exp(-2u): u within 6 roundings, so e within 12 |u| + 2, weighed by e / (1 + e), the sum 1, the
    reciprocal 2 and the product 1. (1e-37: results below the least normal number.)"""
    N, L = hip, hip.lib()
    m, n, k = 512, 2048, 64
    g = gen(act)
    v = torch.linspace(-20, 20, m * n).view(m, n).clone()
    v[:64] = torch.randn(64, n, generator=g) * 0.1
    v[64:128] = torch.randn(64, n, generator=g) * 2
    v[0, :8] = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e30, 3e38, 1.25, -1.25])
    v[1, :2] = torch.tensor([-1e30, -3e38])
    d = N.LinearDesc(m=m, n=n, k=k, dtype=F32, trans_w=1, act=act)
    packed, xd, vd = linear_pack(N, d, torch.zeros(n, k, device="cuda")), torch.zeros(m, k, device="cuda"), v.cuda()
    size = L.spinn_hip_linear_workspace_size(C.byref(d))
    ws, y = workspace(size), torch.empty(m, n, device="cuda")
    N.check(L.spinn_hip_linear(C.byref(d), ptr(xd), ptr(packed), None, ptr(vd), ptr(y), ptr(ws), size, stream()), "linear")
    x, step = v.double(), 2.0 ** -24
    if act == 6:
        ref = x * 0.5 * torch.erfc(-x * 0.5 ** 0.5)
        tol = 3 * step * x.abs()
        tol = torch.where(x < 0, torch.minimum(tol, (10 + x * x) * step * ref.abs()), tol)
    else:
        u = (2 / math.pi) ** 0.5 * (x + 0.044715 * x ** 3)
        share = torch.sigmoid(-2 * u)  # e / (1 + e)
        ref = x * torch.sigmoid(2 * u)
        tol = ref.abs() * step * (4 + (12 * u.abs() + 2) * share)
    assert_close(y, ref, tol + 1e-37 * (1 + x.abs().clamp(max=100)), f"gelu {act}")


def test_linear_values(hip, torch_gpu):
    """Infinities and NaN reach the outputs of their row and column alone; ReLU and SiLU of large
    magnitudes; an empty batch."""
    N, L = hip, hip.lib()
    for m in (4, 70, 600):
        n, k = 128, 64
        g = gen(m)
        x, w = randn(g, m, k, dtype=BF16), randn(g, n, k, dtype=BF16, scale=0.125)
        x[1, 5], x[3, 0] = float("inf"), float("nan")
        w[7, 9] = float("inf")
        d = N.LinearDesc(m=m, n=n, k=k, dtype=BF16, trans_w=1, act=0)
        packed, xd = linear_pack(N, d, w.cuda()), x.cuda()
        y = torch.empty(m, n, device="cuda", dtype=torch.bfloat16)
        N.check(L.spinn_hip_linear(C.byref(d), ptr(xd), ptr(packed), None, None, ptr(y), None, 0, stream()), "linear")
        ref = x.double() @ w.double().t()
        y = y.cpu().double()
        assert torch.equal(y.isnan(), ref.isnan())
        assert torch.equal(torch.where(y.isinf(), y, 0.0), torch.where(ref.isinf(), ref, 0.0))
        big = (torch.randn(m, n, generator=g) * 30000).clamp(-60000, 60000).half()
        d = N.LinearDesc(m=m, n=n, k=k, dtype=F16, trans_w=1, act=3)
        packed, xd = linear_pack(N, d, torch.zeros(n, k, dtype=torch.float16, device="cuda")), torch.zeros(m, k, dtype=torch.float16, device="cuda")
        y, bd = torch.empty(m, n, device="cuda", dtype=torch.float16), big.cuda()
        N.check(L.spinn_hip_linear(C.byref(d), ptr(xd), ptr(packed), None, ptr(bd), ptr(y), None, 0, stream()), "linear")
        ref = torch.nn.functional.silu(big.double()).half()
        assert torch.equal(y.cpu(), ref + 0.0)
    d = N.LinearDesc(m=0, n=n, k=k, dtype=F16, trans_w=1, act=3)
    assert L.spinn_hip_linear(C.byref(d), None, None, None, None, None, None, 0, None) == 0

"""spinn_hip_rope on the GPU against 64 bits; the bounds are derived in promptops.rope_ref."""
import ctypes as C

import pytest
import torch

from tests.decodeops import BF16, F16, F32, NAMES, TORCH, assert_close, gen, ptr, randn, stream
from tests.promptops import rope_frequencies, rope_ref

pytestmark = pytest.mark.gpu

SCALINGS = {"plain": (0, 1.0), "linear": (1, 4.0), "parts": (2, 8.0)}


def desc(N, dtype, heads, dim, rot, inter, scaling="plain", base=10000.0, magnitude=1.0, strides=(0, 0, 0, 0)):
    kind, factor = SCALINGS[scaling]
    return N.RopeDesc(dtype=dtype, heads=heads, head_dim=dim, rot_dim=rot, interleaved=int(inter), scaling=kind, base=base, factor=factor,
                      low=1.0, high=4.0, trained=512, magnitude=magnitude, x_stride=strides[0], x_head_stride=strides[1],
                      y_stride=strides[2], y_head_stride=strides[3])


def table(N, d):
    t = torch.zeros(N.lib().spinn_hip_rope_table_size(C.byref(d)), dtype=torch.uint8, device="cuda")
    N.check(N.lib().spinn_hip_rope_table(C.byref(d), ptr(t), stream()), "table")
    return t


def run(N, d, position, tab, x, y):
    N.check(N.lib().spinn_hip_rope(C.byref(d), position.numel(), ptr(position), ptr(tab), ptr(x), ptr(y), stream()), "rope")


def check(N, dtype, tokens, heads, dim, rot, inter, scaling="plain", in_place=False, pad=0, head_pad=0, offset=0, positions=None, base=10000.0,
          magnitude=1.0, seed=0):
    g = gen(seed + tokens * 7 + dim)
    hs = dim + head_pad
    width = heads * hs + pad
    flat = randn(g, offset + tokens * width, dtype=dtype).cuda()
    x = flat[offset:].view(tokens, width)
    heads_of = lambda t, s: t.as_strided((tokens, heads, dim), (t.stride(0), s, 1))  # noqa: E731
    before = x.clone()
    position = (torch.randint(0, 5000, (tokens,), generator=g) if positions is None else positions).to(torch.int32).cuda()
    if in_place:
        y, ys = x, hs
    else:
        ys = dim + 1 if offset else dim
        y = torch.full((tokens, heads * ys + 3), 7.0, dtype=TORCH[dtype], device="cuda")
    d = desc(N, dtype, heads, dim, rot, inter, scaling, base, magnitude, (x.stride(0), hs, y.stride(0), ys))
    run(N, d, position, table(N, d), x, y)
    kind, factor = SCALINGS[scaling]
    f = rope_frequencies(rot, base, kind, factor, 1.0, 4.0, 512)
    src = heads_of(before, hs).cpu()
    want, tol = rope_ref(src, position.cpu(), f, rot, inter, magnitude, dtype)
    got = heads_of(y, ys).cpu()
    assert torch.equal(got[..., rot:], src[..., rot:])  # copied
    assert_close(got[..., :rot], want[..., :rot], tol[..., :rot], f"rope {NAMES[dtype]} {tokens}x{heads}x{dim}/{rot} {scaling} inter={inter}")
    # nothing else was touched
    mask = torch.ones_like(y, dtype=torch.bool)
    heads_of(mask, ys)[:] = False
    assert torch.equal(y[mask], before[mask] if in_place else torch.full_like(y[mask], 7.0))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("inter", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,dim,rot,in_place", [
    (1, 1, 2, 2, True), (1, 8, 128, 128, True), (5, 20, 128, 128, False), (33, 3, 80, 32, False), (257, 5, 96, 48, True), (3, 7, 66, 66, False),
    (17, 2, 67, 34, False), (9, 2, 67, 34, True), (4, 1, 512, 512, False), (2500, 3, 64, 64, True), (40, 64, 256, 256, False), (6, 5, 33, 30, False)])
def test_layouts(hip, dtype, inter, tokens, heads, dim, rot, in_place):
    check(hip, dtype, tokens, heads, dim, rot, inter, in_place=in_place)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
@pytest.mark.parametrize("inter", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("pad,head_pad,offset", [(8, 0, 0), (5, 0, 0), (0, 3, 0), (64, 16, 1), (1, 1, 3)])
def test_strides_and_alignment(hip, dtype, inter, pad, head_pad, offset):
    for dim, rot in ((64, 64), (80, 40), (35, 18)):
        check(hip, dtype, 19, 3, dim, rot, inter, pad=pad, head_pad=head_pad, offset=offset)
        check(hip, dtype, 19, 3, dim, rot, inter, pad=pad, head_pad=head_pad, offset=offset, in_place=True)


@pytest.mark.parametrize("scaling", list(SCALINGS))
@pytest.mark.parametrize("base", [10000.0, 500000.0, 0.5])
def test_scalings(hip, scaling, base):
    check(hip, F32, 300, 2, 128, 128, False, scaling, base=base, magnitude=1.0 if scaling == "plain" else 1.2079)


def test_far_positions(hip):
    """Positions up to the largest, negative ones, and 0, which turns nothing."""
    far = torch.tensor([0, 1, -1, 4096, 131071, 131072, 1 << 20, -(1 << 20), (1 << 24) + 1, (1 << 30) + 3, 2 ** 31 - 1, -(2 ** 31)])
    for inter in (False, True):
        check(hip, F32, far.numel(), 2, 64, 64, inter, positions=far)
    x = randn(gen(1), 4, 2, 64, dtype=F32).cuda()
    y = torch.zeros_like(x)
    d = desc(hip, F32, 2, 64, 64, False, strides=(128, 64, 128, 64))
    run(hip, d, torch.zeros(4, dtype=torch.int32, device="cuda"), table(hip, d), x, y)
    assert torch.equal(x, y)


def test_there_and_back(hip):
    """Turned by p and then by -p: the input again, up to the roundings of both (twice the bound of one)."""
    g = gen(2)
    x = randn(g, 100, 4, 64, dtype=F32).cuda()
    p = torch.randint(0, 100000, (100,), generator=g).to(torch.int32).cuda()
    d = desc(hip, F32, 4, 64, 64, False, strides=(256, 64, 256, 64))
    tab, y = table(hip, d), x.clone()
    run(hip, d, p, tab, y, y)
    run(hip, d, -p, tab, y, y)
    pair = x.abs() + x.abs().view(100, 4, 2, 32).flip(2).reshape(100, 4, 64)
    assert_close(y, x, 2 * 2.0 ** -21 * pair, "there and back")


def test_special_values(hip):
    """A NaN or an infinity stays in its pair; the copied rest keeps its bits."""
    x = randn(gen(3), 2, 1, 16, dtype=F32).cuda()
    x[0, 0, 3], x[1, 0, 12] = float("nan"), float("inf")
    d = desc(hip, F32, 1, 16, 8, True, strides=(16, 16, 16, 16))
    y = torch.zeros_like(x)
    run(hip, d, torch.tensor([5, 9], dtype=torch.int32, device="cuda"), table(hip, d), x, y)
    assert y[0, 0, 2:4].isnan().all() and y[0, 0, :2].isfinite().all() and y[0, 0, 4:].isfinite().all()
    assert y[1, 0, 12] == float("inf") and torch.equal(y[..., 8:].view(torch.int32), x[..., 8:].view(torch.int32))


def test_many_tokens_over_blocks(hip):
    """Tokens that do not fill the last workgroup, and positions that only the device knows."""
    check(hip, BF16, 20001, 2, 64, 64, False)
    check(hip, F16, 4099, 1, 32, 16, True)

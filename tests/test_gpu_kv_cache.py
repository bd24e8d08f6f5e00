"""The paged key-value cache: spinn_hip_kv_append, spinn_hip_kv_attention, spinn_hip_kv_evict against
their definitions in 64 bits (bounds derived in tests/decodeops.py, attention_ref; copies are exact)."""
import ctypes as C
import math

import pytest
import torch

from tests.decodeops import (BF16, F16, F32, NAMES, TORCH, Cache, assert_close, attention_ref, evict_ref, gen, ptr, randn,
                             stream, workspace)

pytestmark = pytest.mark.gpu


def shifted(x, by):
    """x's elements at an address `by` elements behind an aligned one."""
    return torch.cat([x.new_zeros(by), x.flatten()])[by:].view(x.shape)


def attend(N, c, lengths, heads, scale=None, mask=None, accumulate=False, seed=0, max_len=None, qpad=0, opad=0, lse=True,
           shift=0):
    """One call and its comparison; rows around the outputs have to stay as they were."""
    L, g, t = N.lib(), gen(seed), TORCH[c.dtype]
    S, d, slots = c.seqs, c.dim, c.max_pages * c.page
    scale = 2.0 * d ** -0.5 if scale is None else scale
    max_len = slots if max_len is None else max_len
    q = randn(g, S, heads, d, dtype=c.dtype)
    qd = torch.full((S, heads * d + qpad), float("nan"), dtype=t, device="cuda")
    qd[:, :heads * d] = q.view(S, heads * d).cuda()
    od = torch.full((S, heads * d + opad), 777.0, dtype=t, device="cuda")
    lsed = torch.full((S, heads), 777.0, device="cuda")
    acc = torch.rand(S, c.kv, slots, generator=g)
    accd, outd = acc.cuda(), torch.full((S, c.kv, slots), 777.0, device="cuda")
    kd, vd, td = c.k.cuda(), c.v.cuda(), c.table.cuda()
    if shift:
        qd, od, kd, vd = (shifted(x, shift) for x in (qd, od, kd, vd))
    ld = torch.tensor(lengths, dtype=torch.int32).cuda()
    md = None if mask is None else mask.cuda()
    desc = N.KvAttentionDesc(kv=c.desc(N), heads=heads, max_len=max_len, scale=scale, accumulate=int(accumulate),
                             q_stride=heads * d + qpad, o_stride=heads * d + opad,
                             mask_stride=0 if mask is None else mask.shape[1], acc_stride=slots)
    size = L.spinn_hip_kv_attention_workspace_size(C.byref(desc))
    ws = workspace(size)
    print(f"[attend] {NAMES[c.dtype]} seqs={S} heads={heads}/{c.kv} dim={d} page={c.page} lengths={lengths[:8]} ws={size}", flush=True)
    N.check(L.spinn_hip_kv_attention(C.byref(desc), ptr(qd), ptr(kd), ptr(vd), ptr(td), ptr(ld), ptr(md),
                                     ptr(accd) if accumulate else None, ptr(outd) if accumulate else None, ptr(od),
                                     ptr(lsed) if lse else None, ptr(ws), size, stream()), "spinn_hip_kv_attention")
    torch.cuda.synchronize()
    o, o_tol, lref, l_tol, w, w_tol = attention_ref(c, q, lengths, scale, max_len, mask)
    assert_close(od[:, :heads * d].reshape(S, heads, d), o, o_tol, "o")
    assert (od[:, heads * d:] == 777).all()
    if lse:
        got = lsed.cpu().double()
        assert torch.equal(got == -math.inf, lref == -math.inf)
        assert_close(torch.where(lref == -math.inf, 0.0, got), torch.where(lref == -math.inf, 0.0, lref), l_tol + 1e-37, "lse")
    else:
        assert (lsed == 777).all()
    if accumulate:
        got = outd.cpu()
        for s in range(S):
            n = min(max(lengths[s], 0), max_len)
            assert (got[s, :, n:] == 777).all()
            want = acc[s, :, :n].double() + w[s, :, :n]
            assert_close(got[s, :, :n], want, w_tol[s, :, :n] + 2.0 ** -23 * want, f"weights of sequence {s}")
    return od


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("dim", [1, 3, 4, 5, 7, 8, 9, 20, 32, 33, 64, 80, 96, 100, 127, 128, 129, 160, 251, 256])
def test_attention_dims(hip, torch_gpu, dtype, dim):
    c = Cache(gen(dim), dtype, 3, 2, dim, 16, 100)
    attend(hip, c, [100, 1, 37], heads=4, accumulate=True)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
@pytest.mark.parametrize("page", [1, 3, 8, 16, 20, 48, 128])
def test_attention_pages(hip, torch_gpu, dtype, page):
    """Pages that end inside a tile of slots, and sequences that end inside a page."""
    c = Cache(gen(page), dtype, 4, 2, 64, page, 300)
    attend(hip, c, [300, 129, 31, 16], heads=2, seed=page)


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (6, 2), (16, 1), (17, 1), (40, 2), (128, 1)])
@pytest.mark.parametrize("dtype", [F32, F16], ids=NAMES.get)
def test_attention_head_groups(hip, torch_gpu, dtype, heads, kv):
    c = Cache(gen(heads), dtype, 2, kv, 64, 16, 200)
    attend(hip, c, [200, 77], heads=heads, accumulate=True)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
def test_attention_many_long_heads(hip, torch_gpu, dtype):
    """The most query heads a workgroup takes, at the longest rows: the most that it joins on chip."""
    c = Cache(gen(2), dtype, 1, 2, 256, 16, 500)
    attend(hip, c, [500], heads=32, accumulate=True)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("slots", [1, 2, 31, 32, 33, 127, 128, 129, 255, 257, 1000, 5000])
def test_attention_lengths(hip, torch_gpu, dtype, slots):
    """One sequence, so that longer ones are split over workgroups and joined."""
    c = Cache(gen(slots), dtype, 1, 1, 64, 16, slots)
    attend(hip, c, [slots], heads=2, accumulate=True, seed=slots)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
@pytest.mark.parametrize("seqs,kv,heads,slots", [(70, 1, 2, 900), (130, 3, 3, 700), (1, 5, 10, 3000), (3, 2, 34, 1500), (600, 1, 1, 600)])
def test_attention_ragged_batches(hip, torch_gpu, dtype, seqs, kv, heads, slots):
    """Lengths from nothing to all of it, in no order: rows that lie in one workgroup's share, that several share, and
    shares of several rows; fewer steps than workgroups; more sequences than a wave looks at."""
    g = gen(seqs)
    c = Cache(g, dtype, seqs, kv, 16, 16, slots)
    lengths = (torch.rand(seqs, generator=g) ** 4 * slots).int().tolist()
    lengths[0], lengths[-1] = slots, (0 if seqs > 1 else slots)
    attend(hip, c, lengths, heads=heads, accumulate=True)
    if seqs > 1:
        attend(hip, c, [0] * (seqs - 1) + [5], heads=heads, accumulate=True, seed=1)
        attend(hip, c, [0] * seqs, heads=heads, accumulate=True, seed=2)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("slots,dim,page", [(129, 64, 16), (250, 128, 16), (256, 80, 5), (500, 64, 16), (512, 128, 48), (513, 64, 16)])
def test_attention_short_sequences(hip, torch_gpu, dtype, slots, dim, page):
    """Sequences that fit one workgroup's waves, masked, ragged and empty ones among them."""
    g = gen(slots)
    c = Cache(g, dtype, 5, 2, dim, page, slots)
    mask = (torch.rand(5, c.max_pages * page, generator=g) < 0.8).to(torch.uint8)
    mask[3] = 0
    attend(hip, c, [slots, slots // 2, 1, 100, 0], heads=8, mask=mask, accumulate=True, max_len=slots)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("page", [16, 5])
def test_attention_masks_and_empty_rows(hip, torch_gpu, dtype, page):
    """Padding, scattered holes, rows that the mask empties, lengths of zero, below zero and past max_len;
    what hidden slots hold is infinite or NaN."""
    g = gen(11 + page)
    c = Cache(g, dtype, 6, 2, 64, page, 700)
    slots = c.max_pages * c.page
    mask = torch.ones(6, slots + 3, dtype=torch.uint8)
    mask[0, :200] = 0
    mask[1] = (torch.rand(slots + 3, generator=g) < 0.5).to(torch.uint8) * 255
    mask[2] = 0
    for s in range(3):
        for i in range(slots):
            if not mask[s, i]:
                p = int(c.table[s, i // page])
                c.view(c.k)[p, :, i % page] = float("nan") if i % 2 else float("inf")
                c.view(c.v)[p, :, i % page] = float("nan") if i % 3 else float("-inf")
    attend(hip, c, [700, 650, 300, 0, -5, 10 ** 6], heads=6, mask=mask, accumulate=True, max_len=690)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
@pytest.mark.parametrize("page", [16, 7])
def test_attention_rows_behind_the_end_are_not_used(hip, torch_gpu, dtype, page):
    """Slots behind a sequence's end hold NaN."""
    c = Cache(gen(3), dtype, 3, 2, 64, page, 400)
    lengths = [1, 200, 399]
    for s, n in enumerate(lengths):
        for i in range(n, c.max_pages * page):
            p = int(c.table[s, i // page])
            c.view(c.k)[p, :, i % page] = float("nan")
            c.view(c.v)[p, :, i % page] = float("nan")
    attend(hip, c, lengths, heads=4, accumulate=True)


@pytest.mark.parametrize("dtype", [F32, F16], ids=NAMES.get)
@pytest.mark.parametrize("page", [16, 6])
def test_attention_pages_that_hold_nothing(hip, torch_gpu, dtype, page):
    """Page numbers below 0 and from n_pages on: their slots count as hidden, a sequence of them as empty."""
    c = Cache(gen(4), dtype, 3, 2, 64, page, 300)
    c.table[0, 3], c.table[0, 5] = -1, c.n_pages
    c.table[1, :] = 2 ** 31 - 1
    c.table[2, 0] = -2 ** 31
    attend(hip, c, [300, 250, 290], heads=4, accumulate=True)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
@pytest.mark.parametrize("layout,pad", [("slot", 0), ("slot", 8), ("head", 8), ("head", 3)])
def test_attention_layouts(hip, torch_gpu, dtype, layout, pad):
    """Pages by slot and by head, padded rows, query and output rows inside wider ones."""
    c = Cache(gen(5), dtype, 3, 4, 64, 16, 150, layout=layout, pad=pad)
    attend(hip, c, [150, 90, 5], heads=8, qpad=5, opad=3, lse=False)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("dim,page", [(64, 16), (33, 5), (4, 16)])
def test_attention_unaligned_bases(hip, torch_gpu, dtype, dim, page):
    """Queries, cache and results that start at multiples of their element's size only."""
    c = Cache(gen(dim + page), dtype, 3, 2, dim, page, 200)
    even = attend(hip, c, [200, 0, 77], heads=6, accumulate=True, lse=True)
    odd = attend(hip, c, [200, 0, 77], heads=6, accumulate=True, lse=True, shift=1)
    assert odd.shape == even.shape


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
def test_attention_one_slot_outweighs_the_rest(hip, torch_gpu, dtype):
    """One score 17 above thousands of equal ones: the rest together still weigh 2^-12 or so each way, which fp16
    weights would lose one by one."""
    c = Cache(gen(6), dtype, 1, 1, 64, 16, 6000)
    c.view(c.k)[:] = 0
    c.view(c.k)[int(c.table[0, 100]), 0, 3] = 1.0
    L = 6000
    q = torch.full((1, 1, 64), 17.0 / 64)
    t = TORCH[dtype]
    N, lib = hip, hip.lib()
    desc = N.KvAttentionDesc(kv=c.desc(N), heads=1, max_len=L, scale=1.0, q_stride=64, o_stride=64)
    size = lib.spinn_hip_kv_attention_workspace_size(C.byref(desc))
    ws, o = workspace(size), torch.empty(1, 1, 64, dtype=t, device="cuda")
    qd, kd, vd, td, ld = q.to(t).cuda(), c.k.cuda(), c.v.cuda(), c.table.cuda(), torch.tensor([L], dtype=torch.int32).cuda()
    N.check(lib.spinn_hip_kv_attention(C.byref(desc), ptr(qd), ptr(kd), ptr(vd), ptr(td), ptr(ld), None, None, None, ptr(o),
                                       None, ptr(ws), size, stream()), "attention")
    ref, tol, *_ = attention_ref(c, q.to(t), [L], 1.0, L)
    assert_close(o, ref, tol, "o")


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 5), (256, 16)])
def test_attention_weights_keep_all_bits(hip, torch_gpu, dim, page):
    """Weights 1, p, 1 over values -h, 1, -l, where h + l are the first 16 bits of p in two bf16 numbers: what is left of p is
    the result, below 2^-17. p is off by an exponential's 2^-23 (its argument, at most 0.2, by 2^-25), the three terms' sums and
    their division by three roundings of numbers up to 1 each: 2^-22 of the denominator's 2 to 3 in all."""
    N, L, n = hip, hip.lib(), 100
    c = Cache(gen(dim), BF16, n, 1, dim, page, 16)
    score = (torch.arange(1, n + 1).double() * 2.0 ** -9).bfloat16().double()
    p = torch.exp(-score)
    h = p.bfloat16().double()
    l = (p - h).bfloat16().double()
    for s in range(n):
        for i, (key, value) in enumerate(((score[s], -h[s]), (0.0, 1.0), (score[s], -l[s]))):
            at = int(c.table[s, i // page])
            c.view(c.k)[at, 0, i % page] = 0
            c.view(c.k)[at, 0, i % page, 0] = float(key)
            c.view(c.v)[at, 0, i % page] = float(value)
    q = torch.zeros(n, 1, dim)
    q[:, 0, 0] = 1
    d = N.KvAttentionDesc(kv=c.desc(N), heads=1, max_len=16, scale=1.0, q_stride=dim, o_stride=dim)
    size = L.spinn_hip_kv_attention_workspace_size(C.byref(d))
    ws, o = workspace(size), torch.empty(n, dim, dtype=torch.bfloat16, device="cuda")
    qd, kd, vd, td, ld = q.bfloat16().cuda(), c.k.cuda(), c.v.cuda(), c.table.cuda(), torch.full((n,), 3, dtype=torch.int32).cuda()
    N.check(L.spinn_hip_kv_attention(C.byref(d), ptr(qd), ptr(kd), ptr(vd), ptr(td), ptr(ld), None, None, None, ptr(o), None, ptr(ws),
                                     size, stream()), "attention")
    ref = ((p - h - l) / (2 + p))[:, None].expand(n, dim)
    assert ref.abs().max() > 8 * 2.0 ** -23
    assert_close(o, ref, 2.0 ** -22 / 2 + 2.0 ** -8 * ref.abs(), "what is left of p")


def test_attention_far_pages(hip, torch_gpu):
    """Pages whose offsets pass 32 bits of elements."""
    N, lib = hip, hip.lib()
    far = (1 << 32) + 64
    c = Cache(gen(7), F16, 1, 1, 64, 16, 32, extra=0)
    c.table = torch.tensor([[1, 0]], dtype=torch.int32)
    big = [torch.empty(far + 16 * 64, dtype=torch.float16, device="cuda") for _ in range(2)]
    for b, t in zip(big, (c.k, c.v)):
        b[:1024] = t[0].reshape(-1).cuda()
        b[far:far + 1024] = t[1].reshape(-1).cuda()
    kv = c.desc(N)
    kv.page_stride = far
    desc = N.KvAttentionDesc(kv=kv, heads=2, max_len=32, scale=0.25, q_stride=128, o_stride=128)
    q = randn(gen(8), 1, 2, 64, dtype=F16)
    size = lib.spinn_hip_kv_attention_workspace_size(C.byref(desc))
    ws, o = workspace(size), torch.empty(1, 2, 64, dtype=torch.float16, device="cuda")
    qd, td, ld = q.cuda(), c.table.cuda(), torch.tensor([30], dtype=torch.int32).cuda()
    N.check(lib.spinn_hip_kv_attention(C.byref(desc), ptr(qd), ptr(big[0]), ptr(big[1]), ptr(td), ptr(ld), None, None, None,
                                       ptr(o), None, ptr(ws), size, stream()), "attention")
    ref, tol, *_ = attention_ref(c, q, [30], 0.25, 32)
    assert_close(o, ref, tol, "o")


# ---- append ----

@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("dim,page,layout,pad", [(64, 16, "head", 2), (64, 16, "head", 8), (24, 5, "slot", 0), (33, 5, "slot", 2)])
def test_append(hip, torch_gpu, dtype, dim, page, layout, pad):
    """Tokens of a ragged batch, out of the rows of a fused projection; those outside the cache or on a page that
    holds nothing are skipped, all else stays."""
    N, L, g = hip, hip.lib(), gen(dim)
    c = Cache(g, dtype, 3, 2, dim, page, 40, layout=layout, poison=5.0)
    c.table[1, 1] = -1
    slots, row = c.max_pages * page, 2 * dim
    seq = torch.tensor([0, 0, 2, 1, 1, 3, -1, 0, 2, 2], dtype=torch.int32)
    slot = torch.tensor([0, 39, 7, 3, page, 1, 1, slots, -1, 20], dtype=torch.int32)
    position = torch.arange(100, 110, dtype=torch.int32)
    qkv = randn(g, 10, 3 * row + pad, dtype=dtype)
    acc, pos = torch.rand(3, 2, slots, generator=g), torch.full((3, 2, slots), 9, dtype=torch.int32)
    k0, v0 = c.k.clone(), c.v.clone()
    wa, wp = acc.clone(), pos.clone()
    for t in range(10):
        s, i = int(seq[t]), int(slot[t])
        if not (0 <= s < 3 and 0 <= i < slots) or not 0 <= int(c.table[s, i // page]) < c.n_pages:
            continue
        p = int(c.table[s, i // page])
        c.view(k0)[p, :, i % page] = qkv[t, row:2 * row].view(2, dim)
        c.view(v0)[p, :, i % page] = qkv[t, 2 * row:3 * row].view(2, dim)
        wa[s, :, i], wp[s, :, i] = 0, int(position[t])
    dev = [t.cuda() for t in (seq, slot, position, qkv, c.table, c.k, c.v, acc, pos)]
    sd, od, pd, xd, td, kd, vd, ad, bd = dev
    e = qkv.element_size()
    d = c.desc(N)
    N.check(L.spinn_hip_kv_append(C.byref(d), 10, ptr(sd), ptr(od), ptr(pd), C.c_void_p(xd.data_ptr() + row * e), 3 * row + pad,
                                  C.c_void_p(xd.data_ptr() + 2 * row * e), 3 * row + pad, ptr(td), ptr(kd), ptr(vd), ptr(ad),
                                  ptr(bd), slots, stream()), "append")
    torch.cuda.synchronize()
    assert torch.equal(kd.cpu(), k0) and torch.equal(vd.cpu(), v0)
    assert torch.equal(ad.cpu(), wa) and torch.equal(bd.cpu(), wp)
    # one token per sequence, positions and weights not kept
    slot = torch.tensor([2, 4, 11], dtype=torch.int32).cuda()
    N.check(L.spinn_hip_kv_append(C.byref(d), 3, None, ptr(slot), None, C.c_void_p(xd.data_ptr() + row * e), 3 * row + pad,
                                  C.c_void_p(xd.data_ptr() + 2 * row * e), 3 * row + pad, ptr(td), ptr(kd), ptr(vd), None, None,
                                  0, stream()), "append")
    for s, i in enumerate((2, 4, 11)):
        p = int(c.table[s, i // page])
        c.view(k0)[p, :, i % page] = qkv[s, row:2 * row].view(2, dim)
        c.view(v0)[p, :, i % page] = qkv[s, 2 * row:3 * row].view(2, dim)
    torch.cuda.synchronize()
    assert torch.equal(kd.cpu(), k0) and torch.equal(vd.cpu(), v0)


# ---- eviction ----

def evict(N, c, lengths, acc, pos, next_pos, budget, recent, sinks, max_len=None, alias=True):
    L = N.lib()
    slots = acc.shape[2]
    max_len = slots if max_len is None else max_len
    desc = N.KvEvictDesc(kv=c.desc(N), budget=budget, recent=recent, sinks=sinks, max_len=max_len, acc_stride=slots)
    size = L.spinn_hip_kv_evict_workspace_size(C.byref(desc))
    ws = workspace(size)
    kd, vd, td = c.k.cuda(), c.v.cuda(), c.table.cuda()
    ld, nd = torch.tensor(lengths, dtype=torch.int32).cuda(), torch.tensor(next_pos, dtype=torch.int32).cuda()
    ad, pd = acc.cuda(), pos.cuda()
    ao, po, lo = (ad, pd, ld) if alias else (torch.full_like(ad, 777.0), torch.full_like(pd, 777), torch.full_like(ld, 777))
    print(f"[evict] {NAMES[c.dtype]} lengths={lengths[:6]} budget={budget} recent={recent} sinks={sinks} ws={size}", flush=True)
    N.check(L.spinn_hip_kv_evict(C.byref(desc), ptr(td), ptr(ld), ptr(nd), ptr(ad), ptr(pd), ptr(ao), ptr(po), ptr(lo),
                                 ptr(kd), ptr(vd), ptr(ws), size, stream()), "evict")
    torch.cuda.synchronize()
    moves, wa, wp, wl = evict_ref(c, lengths, next_pos, acc, pos, budget, recent, sinks, max_len)
    assert lo.tolist() == wl
    behind_a, behind_p = (acc, pos) if alias else (torch.full_like(acc, 777.0), torch.full_like(pos, 777))
    for (s, h), a in wa.items():
        n = len(a)
        assert torch.equal(ao[s, h, :n].cpu().nan_to_num(nan=-7.0), torch.tensor(a).nan_to_num(nan=-7.0)), (s, h)
        assert po[s, h, :n].tolist() == wp[s, h], (s, h)
        assert torch.equal(ao[s, h, n:].cpu().nan_to_num(nan=-7.0), behind_a[s, h, n:].nan_to_num(nan=-7.0))
        assert torch.equal(po[s, h, n:].cpu(), behind_p[s, h, n:])
    for t, got in ((c.k, kd), (c.v, vd)):
        want, old = t.clone(), t.clone()
        for s, h, frm, to in moves:
            p, q = int(c.table[s, frm // c.page]), int(c.table[s, to // c.page])
            if 0 <= p < c.n_pages and 0 <= q < c.n_pages:
                c.view(want)[q, h, to % c.page] = c.view(old)[p, h, frm % c.page]
        assert torch.equal(got.cpu().nan_to_num(nan=-7.0), want.nan_to_num(nan=-7.0))


def _evictable(seed, dtype, seqs, kv, dim, page, slots, **kw):
    g = gen(seed)
    c = Cache(g, dtype, seqs, kv, dim, page, slots, **kw)
    n = c.max_pages * page
    acc = torch.exp(2 * torch.randn(seqs, kv, n, generator=g))
    pos = torch.arange(n, dtype=torch.int32).expand(seqs, kv, n).contiguous()
    return g, c, acc, pos


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("dim,page,layout,pad", [(64, 16, "head", 0), (33, 5, "head", 0), (40, 1, "slot", 0), (64, 16, "slot", 3)])
def test_evict(hip, torch_gpu, dtype, dim, page, layout, pad):
    g, c, acc, pos = _evictable(dim + page, dtype, 4, 2, dim, page, 300, layout=layout, pad=pad)
    evict(hip, c, [300, 120, 119, 211], acc, pos, [300, 120, 119, 211], 120, 30, 4)


@pytest.mark.parametrize("alias", [True, False])
@pytest.mark.parametrize("budget,recent,sinks", [(0, 0, 0), (1, 0, 0), (1, 1, 0), (50, 50, 0), (50, 80, 4), (299, 10, 4), (300, 10, 4),
                                                 (400, 10, 4), (128, 0, 0), (128, 0, 1000)])
def test_evict_budgets(hip, torch_gpu, budget, recent, sinks, alias):
    """Budgets of nothing, one, everything and more; more safe tokens than the budget holds (the lower slots stay)."""
    g, c, acc, pos = _evictable(budget, F16, 3, 2, 32, 16, 300)
    evict(hip, c, [300, 299, 7], acc, pos, [300, 299, 7], budget, recent, sinks, alias=alias)


@pytest.mark.parametrize("slots", [1, 2, 1023, 1025, 9000, 20000])
def test_evict_lengths(hip, torch_gpu, slots):
    """Rows around a step of the selection, and longer than what it holds on chip."""
    g, c, acc, pos = _evictable(slots, F16, 1, 1, 8, 16, slots)
    evict(hip, c, [slots], acc, pos, [slots], max(1, slots // 3), slots // 10, 2)


def test_evict_equal_and_odd_weights(hip, torch_gpu):
    """Equal weights (the lower slot stays), zeros of both signs, infinities, NaN; slots in no order of position;
    lengths of zero, below zero and past max_len; a page that holds nothing."""
    g, c, acc, pos = _evictable(5, BF16, 6, 2, 16, 4, 600)
    n = acc.shape[2]
    acc[0] = 1.0
    acc[1] = torch.randint(0, 4, (2, n), generator=g).float()
    acc[2] = torch.where(torch.rand(2, n, generator=g) < 0.5, 0.0, -0.0)
    acc[3, :, ::3], acc[3, :, 1::7], acc[3, :, 2::11] = math.nan, math.inf, -math.inf
    pos = torch.stack([torch.randperm(n, generator=g) for _ in range(12)]).view(6, 2, n).to(torch.int32)
    c.table[1, 20] = -1
    c.table[1, 100] = c.n_pages + 3
    evict(hip, c, [600, 600, 600, 600, 0, 10 ** 6], acc, pos, [600, 580, 600, 610, 3, 600], 200, 64, 4, max_len=590)
    evict(hip, c, [-3, 201, 200, 199, 590, 300], acc, pos, [600, 580, 600, 610, -2 ** 31, 2 ** 31 - 1], 200, 64, 0)


@pytest.mark.parametrize("seqs,max_len,budget", [(256, 9000, 4500), (2048, 131072, 65536)])
def test_evict_many_rows_of_great_capacity(hip, torch_gpu, seqs, max_len, budget):
    """Sizes of many long rows, of which few are in use: more shares of moves than one launch has workgroups of 256 threads.
    The others are empty and their pages hold nothing."""
    N, L, kv, page = hip, hip.lib(), 8, 16
    used = [3, seqs - 2]
    c = Cache(gen(seqs), F16, 2, kv, 8, page, max_len)
    n, pages = max_len, c.max_pages
    table = torch.full((seqs, pages), -1, dtype=torch.int32, device="cuda")
    table[used] = c.table.cuda()
    g = gen(1)
    acc = torch.empty(seqs, kv, n, device="cuda")
    pos = torch.empty(seqs, kv, n, dtype=torch.int32, device="cuda")
    w, p = torch.exp(torch.randn(2, kv, n, generator=g)), torch.arange(n, dtype=torch.int32).expand(2, kv, n)
    acc[used], pos[used] = w.cuda(), p.cuda()
    lengths = torch.zeros(seqs, dtype=torch.int32, device="cuda")
    lengths[used] = torch.tensor([n, n - 11], dtype=torch.int32).cuda()
    desc = c.desc(N)
    desc.seqs = seqs
    d = N.KvEvictDesc(kv=desc, budget=budget, recent=100, sinks=4, max_len=n, acc_stride=n)
    size = L.spinn_hip_kv_evict_workspace_size(C.byref(d))
    ws, kd, vd, next_pos = torch.empty(size, dtype=torch.uint8, device="cuda"), c.k.cuda(), c.v.cuda(), lengths.clone()
    N.check(L.spinn_hip_kv_evict(C.byref(d), ptr(table), ptr(lengths), ptr(next_pos), ptr(acc), ptr(pos), ptr(acc), ptr(pos),
                                 ptr(lengths), ptr(kd), ptr(vd), ptr(ws), size, stream()), "evict")
    assert lengths.tolist() == [budget if s in used else 0 for s in range(seqs)]
    want = {id(t): t.clone() for t in (c.k, c.v)}
    for s, length in enumerate((n, n - 11)):
        key = w[s, :, :length].clone()
        key[:, :4] = key[:, length - 100:] = math.inf
        order = torch.sort(key, dim=1, descending=True, stable=True)[1]
        for h in range(kv):
            kept = torch.sort(order[h, :budget])[0]
            to = torch.ones(budget, dtype=torch.bool)
            to[kept[kept < budget]] = False
            to, frm, source = torch.nonzero(to)[:, 0], kept[kept >= budget], torch.arange(budget)
            source[to] = frm
            assert torch.equal(acc[used[s], h, :budget].cpu(), w[s, h, source])
            assert torch.equal(pos[used[s], h, :budget].cpu(), source.to(torch.int32))
            for t in (c.k, c.v):
                c.view(want[id(t)])[c.table[s, to // page].long(), h, to % page] = c.view(t)[c.table[s, frm // page].long(), h, frm % page]
    for t, got in ((c.k, kd), (c.v, vd)):
        assert torch.equal(got.cpu().nan_to_num(nan=-7.0), want[id(t)].nan_to_num(nan=-7.0))


def test_evict_twice(hip, torch_gpu):
    """Evict, append, evict again: slots are out of order by then, and the positions carry on."""
    N, L = hip, hip.lib()
    g, c, acc, pos = _evictable(9, F32, 2, 2, 32, 16, 100)
    lengths, nxt = [100, 90], [100, 90]
    for step in range(3):
        moves, wa, wp, wl = evict_ref(c, lengths, nxt, acc, pos, 40, 10, 2, 100)
        evict(hip, c, lengths, acc, pos, nxt, 40, 10, 2, max_len=100)
        for t in (c.k, c.v):
            old = t.clone()
            for s, h, frm, to in moves:
                c.view(t)[int(c.table[s, to // 16]), h, to % 16] = c.view(old)[int(c.table[s, frm // 16]), h, frm % 16]
        for (s, h), a in wa.items():
            acc[s, h, :len(a)], pos[s, h, :len(a)] = torch.tensor(a), torch.tensor(wp[s, h], dtype=torch.int32)
        # 15 tokens on
        for s in range(2):
            pos[s, :, 40:55] = torch.arange(nxt[s], nxt[s] + 15, dtype=torch.int32)
            acc[s, :, 40:55] = torch.rand(2, 15, generator=g)
        lengths, nxt = [55, 55], [nxt[0] + 15, nxt[1] + 15]

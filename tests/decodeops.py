"""Descriptors, device tensors and 64-bit references of the decoding step's operators (test helper)."""
from __future__ import annotations

import ctypes as C
import math

import torch

F32, F16, BF16 = 1, 10, 16  # ENNF_TYPE_*
TORCH = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}  # of a rounding, relative to the value
NAMES = {F32: "fp32", F16: "fp16", BF16: "bf16"}
ACTS = {0: lambda v: v, 1: torch.relu, 3: torch.nn.functional.silu, 6: torch.nn.functional.gelu,
        7: lambda v: torch.nn.functional.gelu(v, approximate="tanh")}


def ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(TORCH[dtype])


def workspace(size, fill=0xA5):
    """A workspace of exactly `size` bytes that starts dirty (none for 0)."""
    return torch.full((size,), fill, device="cuda", dtype=torch.uint8) if size else None


def assert_close(y, ref, tol, what):
    """|y - ref| <= tol, element by element (tensors in 64 bits); prints the worst share of the bound."""
    y, ref, tol = y.double().cpu(), ref.double().cpu(), tol.double().cpu()
    assert y.shape == ref.shape, (what, y.shape, ref.shape)
    assert torch.isfinite(y).all(), f"{what}: non-finite output"
    share = float(((y - ref).abs() / tol.clamp(min=1e-300)).max()) if y.numel() else 0.0
    print(f"[bound] {what}: {share:.3f} of the bound", flush=True)
    assert share <= 1.0, f"{what}: {share:.3f} times the bound"


# ---- linear ----

def linear_pack(N, d, w):
    L = N.lib()
    size = L.spinn_hip_linear_packed_size(C.byref(d))
    assert size > 0
    packed = torch.full((size,), 0xA5, device="cuda", dtype=torch.uint8)
    N.check(L.spinn_hip_linear_pack_weights(C.byref(d), ptr(w), ptr(packed), stream()), "pack")
    return packed


def linear_ref(x, w, trans_w, bias, res, act, dtype):
    """(y, bound) in 64 bits. The bound counts: K + 4 roundings of an fp32 sum, each at most 2^-24 of
    the sum of the terms' magnitudes, twice (a matrix instruction may round inside, too); activations'
    slopes of at most 1.13 and their own evaluation, 2^-19 of their argument; the result's rounding."""
    x, w = x.double(), w.double()
    w = w.t() if trans_w else w
    v, s = x @ w, x.abs() @ w.abs()
    for t in (bias, res):
        if t is not None:
            v, s = v + t.double(), s + t.double().abs()
    y = ACTS[act](v)
    sums = 2 * (x.shape[1] + 4) * 2.0 ** -24 * s
    return y, 1.13 * sums + 2.0 ** -19 * v.abs() * (act not in (0, 1)) + HALF_STEP[dtype] * (y.abs() + 1.13 * sums) + 1e-37


# ---- paged cache ----

class Cache:
    """A paged cache on the CPU: random rows in randomly placed pages, the unused ones poisoned."""

    def __init__(self, g, dtype, seqs, kv, dim, page, slots, extra=2, layout="head", pad=0, poison=float("nan")):
        self.dtype, self.seqs, self.kv, self.dim, self.page = dtype, seqs, kv, dim, page
        self.max_pages = max(1, -(-slots // page))
        self.n_pages = seqs * self.max_pages + extra
        order = torch.randperm(self.n_pages, generator=g)
        self.table = order[:seqs * self.max_pages].to(torch.int32).view(seqs, self.max_pages)
        row = dim + pad
        # "head": [page][head][slot][row], "slot": [page][slot][head][row]
        shape = (self.n_pages, kv, page, row) if layout == "head" else (self.n_pages, page, kv, row)
        self.layout = layout
        self.k, self.v = (torch.full(shape, poison).to(TORCH[dtype]) for _ in range(2))
        for t in (self.k, self.v):
            self.view(t)[self.table.view(-1).long()] = randn(g, seqs * self.max_pages, kv, page, dim, dtype=dtype)
        st = self.view(self.k).stride()
        self.strides = (st[0], st[1], st[2])

    def view(self, t):
        """[page, head, slot, dim] view of an array of pages."""
        t = t if self.layout == "head" else t.transpose(1, 2)
        return t[..., :self.dim]

    def desc(self, N):
        return N.KvDesc(dtype=self.dtype, seqs=self.seqs, kv_heads=self.kv, head_dim=self.dim, page_size=self.page,
                        n_pages=self.n_pages, max_pages=self.max_pages, page_stride=self.strides[0],
                        head_stride=self.strides[1], slot_stride=self.strides[2])

    def rows(self, t, s, n):
        """[kv, n, dim] of the first n slots of sequence s, and which of them lie in a page."""
        pages = self.table[s].long()
        ok = (pages >= 0) & (pages < self.n_pages)
        r = self.view(t)[pages.clamp(0, self.n_pages - 1)]  # [pages, kv, page, dim]
        r = r.transpose(0, 1).reshape(self.kv, self.max_pages * self.page, self.dim)[:, :n]
        return r, ok.repeat_interleave(self.page)[:n]


def attention_ref(c, q, lengths, scale, max_len, mask=None):
    """Per (sequence, head): o, lse, and bounds; per (sequence, kv head, slot) the added weight and its bound.

    Scores are fp32 sums of head_dim products: off by e = 2 (dim + 4) 2^-24 sum|q_i k_i| scale at most
    (as in linear_ref) plus their rounding to base 2, 2^-22 of themselves; a weight by 2 e (its own and the maximum's), an exponential's
    2^-21, the parts it is multiplied in, 2^-16 (bf16) or 2^-20 (fp16, least number 2^-39 of the
    largest weight), and the sum of n weights, (n/16 + 64) 2^-23."""
    group = q.shape[1] // c.kv
    S, H, d = q.shape
    slots = c.max_pages * c.page
    o, lse = torch.zeros(S, H, d, dtype=torch.float64), torch.full((S, H), -math.inf, dtype=torch.float64)
    o_tol, lse_tol = torch.zeros_like(o), torch.zeros_like(lse)
    w, w_tol = torch.zeros(S, c.kv, slots, dtype=torch.float64), torch.zeros(S, c.kv, slots, dtype=torch.float64)
    parts = {F32: 0.0, F16: 2.0 ** -20, BF16: 2.0 ** -16}[c.dtype]
    for s in range(S):
        n = min(max(int(lengths[s]), 0), max_len)
        if n == 0:
            continue
        k, ok = c.rows(c.k, s, n)
        v, _ = c.rows(c.v, s, n)
        seen = ok.clone()
        if mask is not None:
            seen &= mask[s, :n] != 0
        if not seen.any():
            continue
        for h in range(H):
            kk, vv = k[h // group].double(), v[h // group].double()
            kk, vv = torch.where(seen[:, None], kk, 0.0), torch.where(seen[:, None], vv, 0.0)
            qq = q[s, h].double()
            sc = scale * (kk @ qq)
            e = float((2 * (d + 4) * 2.0 ** -24 * abs(scale) * (kk.abs() @ qq.abs()) + 2.0 ** -22 * sc.abs()).max())
            p = torch.softmax(torch.where(seen, sc, -math.inf), 0)
            rel = 2 * e + 2.0 ** -21 + (n / 16 + 64) * 2.0 ** -23
            o[s, h] = p @ vv
            # the fp16 parts' least number against the row's largest weight, for every slot
            small = n * 2.0 ** -38 * float(p.max()) if c.dtype == F16 else 0.0
            o_tol[s, h] = (2 * rel + parts) * (p @ vv.abs()) + small * float(vv.abs().max())
            lse[s, h] = torch.logsumexp(torch.where(seen, sc, -math.inf), 0)
            lse_tol[s, h] = rel + 2.0 ** -20 * (1 + abs(float(lse[s, h])))
            w[s, h // group, :n] += p
            w_tol[s, h // group, :n] += 2 * rel * p + 1e-37
    o_tol += HALF_STEP[c.dtype] * (o.abs() + o_tol) + 1e-37
    return o, o_tol, lse, lse_tol, w, w_tol


def evict_ref(c, lengths, next_pos, acc, pos, budget, recent, sinks, max_len):
    """Moves by the definition, slot by slot: ([(seq, head, from, to)], acc, pos, lengths) after it."""
    moves, acc_out, pos_out, len_out = [], {}, {}, []
    for s in range(c.seqs):
        n = min(max(int(lengths[s]), 0), max_len)
        left = min(n, budget)
        len_out.append(left)
        for h in range(c.kv):
            a, p = acc[s, h, :n].tolist(), pos[s, h, :n].tolist()

            def key(i):
                safe = p[i] < sinks or p[i] >= int(next_pos[s]) - recent
                nan = a[i] != a[i]
                return (not safe, nan and not safe, 0.0 if safe or nan else -a[i], i)

            kept = sorted(sorted(range(n), key=key)[:left])
            holes = [i for i in range(left) if i not in set(kept)]
            movers = [i for i in kept if i >= left]
            assert len(holes) == len(movers)
            na, np_ = a[:left], p[:left]
            for to, frm in zip(holes, movers):
                moves.append((s, h, frm, to))
                na[to], np_[to] = a[frm], p[frm]
            acc_out[s, h], pos_out[s, h] = na, np_
    return moves, acc_out, pos_out, len_out


# ---- beams ----

def beam_ref(logits, scores, finished, end, k):
    """(scores, parents, tokens) by a stable sort of 64-bit keys."""
    b, w, v = logits.shape
    big = torch.finfo(torch.float32).max
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x).clamp(max=big)
    sc = torch.where(scores.isnan(), -math.inf, scores.double()).clamp(max=big)
    lse = torch.logsumexp(x, 2, keepdim=True)
    key = sc[:, :, None] + torch.where(x == -math.inf, -math.inf, x - torch.where(lse == -math.inf, 0.0, lse))
    if finished is not None:
        only = torch.full((v,), -math.inf, dtype=torch.float64)
        only[end] = 0.0
        key = torch.where(finished[:, :, None] != 0, sc[:, :, None] + only, key)
    key = torch.where(key.isnan(), -math.inf, key).reshape(b, w * v)
    val, at = torch.sort(key, dim=1, descending=True, stable=True)
    return val[:, :k], (at[:, :k] // v).int(), (at[:, :k] % v).int()

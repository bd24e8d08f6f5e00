"""Descriptors and 64-bit references of the operators around a prompt (test helper)."""
from __future__ import annotations

import ctypes as C
import math

import torch

from tests.decodeops import F16, F32, HALF_STEP, TORCH, ptr, randn, stream, workspace


# ---- pages ----

def assign_ref(new, lengths, nxt, held, free, count, table, page, max_tokens):
    """The definition, request by request. Lists; `free` and `table` are changed in place."""
    seqs, row = len(new), len(table[0])
    lengths, nxt = [max(v, 0) for v in lengths], [max(v, 0) for v in nxt]
    held = [min(max(v, 0), row) for v in held]
    count = min(max(count, 0), len(free))
    for s in range(seqs):
        if new[s] == -1:
            for p in table[s][:held[s]]:
                if count < len(free):
                    free[count] = p
                    count += 1
    total, asked, top = 0, 0, count
    starts, served, where = [], [], []
    for s in range(seqs):
        add = max(new[s], 0)
        starts.append(min(total, max_tokens))
        total += add
        fits = new[s] >= -1 and (add == 0 or (lengths[s] + add <= page * row and total <= max_tokens))
        need = max(0, -(-(lengths[s] + add) // page) - held[s]) if fits and add else 0
        asked += need
        ok = fits and (need == 0 or asked <= top)
        served.append(int(ok))
        for i in range(min(add, max_tokens - len(where))):
            where.append((s, lengths[s] + i, nxt[s] + i) if ok else (-1, -1, 0))
        if new[s] == -1:
            lengths[s] = nxt[s] = held[s] = 0
        elif ok:
            for _ in range(need):
                count -= 1
                table[s][held[s]] = free[count]
                held[s] += 1
            lengths[s] += add
            nxt[s] += add
    starts.append(min(total, max_tokens))
    where += [(-1, -1, 0)] * (max_tokens - len(where))
    return dict(lengths=lengths, next=nxt, held=held, count=[count], starts=starts, served=served, seq=[w[0] for w in where],
                slot=[w[1] for w in where], position=[w[2] for w in where])


# ---- rotary positions ----

def rope_frequencies(rot, base, scaling, factor, low, high, trained):
    i = torch.arange(rot // 2, dtype=torch.float64)
    f = torch.tensor(base, dtype=torch.float64) ** (-2 * i / rot)
    if scaling == 1:
        f = f / factor
    elif scaling == 2:
        t = ((trained * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = t * f + (1 - t) * f / factor
    return f


def rope_ref(x, position, f, rot, interleaved, magnitude, dtype):
    """(y, bound): x [tokens, heads, dim]. Sines and cosines in fp32 are off by 6e-8 (their own rounding and that of the angle
    within a quarter turn, 2^-24 each, and the polynomials' 4e-9) and by the angle's error: 2^-32 of a turn and, for the frequencies' own
    rounding in 64 bits, 2^-50 of the angle. Then the magnitude's rounding and two products' and one sum's: 2^-22 of |x_a| + |x_b| in all."""
    x = x.double()
    angle = position.double()[:, None] * f
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    y = x.clone()
    half = rot // 2
    a = x[..., 0:rot:2] if interleaved else x[..., :half]
    b = x[..., 1:rot:2] if interleaved else x[..., half:rot]
    ya, yb = magnitude * (c * a - s * b), magnitude * (s * a + c * b)
    off = (2.0 ** -22 + 2 * math.pi * 2.0 ** -32 + 2.0 ** -50 * angle.abs())[:, None] * (a.abs() + b.abs()) * abs(magnitude)
    tol = torch.zeros_like(x)
    if interleaved:
        y[..., 0:rot:2], y[..., 1:rot:2] = ya, yb
        tol[..., 0:rot:2] = tol[..., 1:rot:2] = off
    else:
        y[..., :half], y[..., half:rot] = ya, yb
        tol[..., :half] = tol[..., half:rot] = off
    tol[..., :rot] += HALF_STEP[dtype] * (y[..., :rot].abs() + tol[..., :rot]) + 2.0 ** -25 * (dtype == F16) + 1e-37
    return y, tol


# ---- attention ----

def prompt_ref(q, k, v, starts, kv_starts, heads, kv_heads, scale, causal, dtype):
    """(o, bound, lse, bound) of packed rows q [rows, heads, dim], k and v [rows, kv heads, dim]; rows outside every
    sequence are NaN in o.

    A score is an fp32 sum of dim products, off by e = 2 (dim + 4) 2^-24 sum|q_i k_i| |scale| and 2^-22 of itself for base 2
    (as in attention_ref); a weight by 2 e, an exponential's 2^-21 and, in 16-bit types, its own rounding to the type, half
    a step (fp16: 2^-32 of the row's largest weight at least, its least number's half); the sums of n weights by (n + 64) 2^-24
    and, in the products, 2 (n + 64) 2^-24 of the magnitudes' sum."""
    rows, dim = q.shape[0], q.shape[2]
    o = torch.full((rows, heads, dim), math.nan, dtype=torch.float64)
    lse = torch.full((rows, heads), math.nan, dtype=torch.float64)
    o_tol, lse_tol = torch.zeros_like(o), torch.zeros_like(lse)
    group = heads // kv_heads
    for a, b, c, d in zip(starts, starts[1:], kv_starts, kv_starts[1:]):
        nq, nk = b - a, d - c
        if nq <= 0:
            continue
        o[a:b], lse[a:b] = 0, -math.inf
        if nk <= 0:
            continue
        seen = torch.arange(nk) <= (torch.arange(nq)[:, None] + nk - nq) if causal else torch.ones(nq, nk, dtype=torch.bool)
        some = seen.any(1)
        for h in range(heads):
            qq, kk, vv = q[a:b, h].double(), k[c:d, h // group].double(), v[c:d, h // group].double()
            kt = kk.t().contiguous()
            sc = scale * (qq @ kt)
            e = 2 * (dim + 4) * 2.0 ** -24 * abs(scale) * (qq.abs() @ kt.abs()) + 2.0 ** -22 * sc.abs()
            e = torch.where(seen, e, 0.0).amax(1, keepdim=True)
            sc = sc.masked_fill(~seen, -math.inf)
            p = torch.where(some[:, None], torch.softmax(sc, 1), 0.0).nan_to_num(0.0)
            part = 0.0 if dtype == F32 else HALF_STEP[dtype]
            rel = 2 * e + 2.0 ** -21 + 3 * (nk + 64) * 2.0 ** -24
            o[a:b, h] = p @ vv
            o_tol[a:b, h] = (2 * rel + part) * (p @ vv.abs())
            if dtype == F16:
                o_tol[a:b, h] += 2.0 ** -32 * p.amax(1, keepdim=True) * (seen.double() @ vv.abs())
            lse[a:b, h] = torch.logsumexp(sc, 1)
            lse_tol[a:b, h] = rel[:, 0] + 2.0 ** -20 * (1 + lse[a:b, h].abs().nan_to_num(0.0, 0.0, 0.0))
    o_tol += HALF_STEP[dtype] * (o.abs().nan_to_num(0.0) + o_tol) + 2.0 ** -25 * (dtype == F16) + 1e-37
    return o, o_tol, lse, lse_tol


class Prompt:
    """Packed rows with gaps around them (`lead` rows before, `tail` behind) in wider rows of `pad` more elements, poisoned."""

    def __init__(self, g, dtype, lens, heads, kv, dim, kv_lens=None, pad=0, lead=0, tail=0, offset=0, fused=False):
        self.dtype, self.heads, self.kv, self.dim = dtype, heads, kv, dim
        starts = lambda n: [lead + sum(n[:i]) for i in range(len(n) + 1)]  # noqa: E731
        self.starts = starts(lens)
        self.kv_starts = self.starts if kv_lens is None else starts(kv_lens)
        self.rows, self.kv_rows = self.starts[-1] + tail, self.kv_starts[-1] + tail
        t, dev = TORCH[dtype], "cuda"

        def place(rows, width, used):
            flat = torch.full((offset + rows * (width + pad),), math.nan, dtype=t, device=dev)
            view = flat[offset:].view(rows, width + pad)[:, :width]
            body = randn(g, used[-1] - used[0], width, dtype=dtype).to(dev)
            view[used[0]:used[-1]] = body
            return view

        if fused:
            rows = place(self.rows, (heads + 2 * kv) * dim, self.starts)
            self.q, self.k, self.v = rows[:, :heads * dim], rows[:, heads * dim:(heads + kv) * dim], rows[:, (heads + kv) * dim:]
        else:
            self.q = place(self.rows, heads * dim, self.starts)
            self.k, self.v = (place(self.kv_rows, kv * dim, self.kv_starts) for _ in range(2))
        self.o = torch.full((offset + self.rows * (heads * dim + pad),), 7.0, dtype=t, device=dev)[offset:].view(self.rows, -1)[:, :heads * dim]
        self.lse = torch.full((self.rows, heads), 7.0, device=dev)

    def run(self, N, scale, causal, lse=True, starts=None, kv_starts="same"):
        d = N.PromptAttentionDesc(dtype=self.dtype, seqs=len(self.starts) - 1, heads=self.heads, kv_heads=self.kv, head_dim=self.dim,
                                  causal=causal, q_rows=self.rows, kv_rows=self.kv_rows, scale=scale, q_stride=self.q.stride(0),
                                  k_stride=self.k.stride(0), v_stride=self.v.stride(0), o_stride=self.o.stride(0))
        L = N.lib()
        size = L.spinn_hip_prompt_attention_workspace_size(C.byref(d))
        self.ws = workspace(size)
        self.dev_starts = torch.tensor(self.starts if starts is None else starts, dtype=torch.int32, device="cuda")
        self.dev_kv = None if self.kv_starts is self.starts else torch.tensor(self.kv_starts, dtype=torch.int32, device="cuda")
        N.check(L.spinn_hip_prompt_attention(C.byref(d), ptr(self.q), ptr(self.k), ptr(self.v), ptr(self.dev_starts), ptr(self.dev_kv),
                                             ptr(self.o), ptr(self.lse) if lse else None, ptr(self.ws), size, stream()), "prompt")

    def ref(self, scale, causal):
        shape = lambda t, h: t.cpu().reshape(t.shape[0], h, self.dim)  # noqa: E731
        return prompt_ref(shape(self.q, self.heads), shape(self.k, self.kv), shape(self.v, self.kv), self.starts, self.kv_starts,
                          self.heads, self.kv, scale, causal, self.dtype)


# ---- 8-bit linear layers ----

def quantize_ref(x):
    """(values, scales) by the definition, in 64 bits: scales rounded to fp32, quotients to the nearest integer, ties to even."""
    x = x.double()
    bad = ~torch.isfinite(x).all(1)
    top = torch.where(torch.isfinite(x), x, 0.0).abs().amax(1)
    scale = (top / 127).float()
    s = scale.double()[:, None]
    q = torch.where(s > 0, torch.round(torch.where(torch.isfinite(x), x, 0.0) / torch.where(s > 0, s, 1.0)), 0.0).clamp(-127, 127)
    q[bad] = 0
    scale[bad] = math.nan
    return q.to(torch.int8), scale

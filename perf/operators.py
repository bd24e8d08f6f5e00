"""The operators of a decoding step whose speed counts, as plain torch and through the C ABI.

Kinds of case, each a call that a program which generates with this framework makes:

  linear  y = act(x w^T + bias + residual) through spinn_hip_linear, weights packed beforehand
  attend  one new token of every sequence over a paged key-value cache through spinn_hip_kv_attention, with the
          weights that each slot received added up where the cache is evicted from later
  evict   a cache cut to its budget by those weights through spinn_hip_kv_evict
  beam    the next beams out of all beams and the vocabulary through spinn_hip_beam_select, and the beams' states
          reordered after them through spinn_hip_beam_reorder
"""
import ctypes as C
import math

import torch

own = False  # False: run() computes the plain forms; True: run() calls the framework

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
CODES = {"fp32": 1, "fp16": 10, "bf16": 16}  # ENNF_TYPE_*
ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")


def linear(dtype, m, n, k, act="none", bias=True, residual=False, trans_w=1, pad=0):
    return {"op": "linear", "dtype": dtype, "m": m, "n": n, "k": k, "act": act, "bias": bias, "residual": residual,
            "trans_w": trans_w, "pad": pad}


def attend(dtype, seqs, heads, kv_heads, dim, page, min_len, max_len, mask=False, weights=False):
    return {"op": "attend", "dtype": dtype, "seqs": seqs, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "min_len": min_len, "max_len": max_len, "mask": mask, "weights": weights}


def evict(dtype, seqs, kv_heads, dim, page, min_len, max_len, budget, recent, sinks=4):
    return {"op": "evict", "dtype": dtype, "seqs": seqs, "kv_heads": kv_heads, "dim": dim, "page": page,
            "min_len": min_len, "max_len": max_len, "budget": budget, "recent": recent, "sinks": sinks}


def beam(dtype, batch, beams, vocab, k, state, finished=False):
    return {"op": "beam", "dtype": dtype, "batch": batch, "beams": beams, "vocab": vocab, "k": k, "state": state,
            "finished": finished}


def listed():
    named = [
        # one token's projection back into the residual stream: a weight matrix read for a single row
        ("linear_1x4096x4096_bf16", linear("bf16", 1, 4096, 4096, residual=True)),
        # the wide layer for a small batch of sequences, no multiple of a tile
        ("linear_33x8192x2048_fp16", linear("fp16", 33, 8192, 2048, "gelu_tanh")),
        # an ordinary MLP layer over the tokens of a batch of images, in the graphs' own type
        ("linear_1568x2048x512_fp32", linear("fp32", 1568, 2048, 512, "gelu")),
        # a whole prompt through the wide layer, its weights as a MatMul node holds them
        ("linear_4096x8192x4096_bf16", linear("bf16", 4096, 8192, 4096, "silu", trans_w=0)),
        # the smallest step: a single short sequence, where latency is all
        ("attend_1x500_fp16", attend("fp16", 1, 16, 4, 64, 16, 500, 500)),
        # a serving batch of ragged sequences
        ("attend_32x8000_bf16", attend("bf16", 32, 32, 8, 128, 16, 37, 8000)),
        # one sequence over a whole book: work only from splitting its length
        ("attend_1x131001_bf16", attend("bf16", 1, 32, 8, 128, 64, 131001, 131001)),
        # heads of their own keys, padded sequences, weights accumulated for the eviction
        ("attend_16x2000_fp32_weights", attend("fp32", 16, 16, 16, 80, 32, 1500, 2000, mask=True, weights=True)),
        # one sequence a few tokens over its budget, during generation
        ("evict_1x520_fp16", evict("fp16", 1, 4, 64, 16, 520, 520, 512, 64)),
        # a batch cut to half after its prompts
        ("evict_16x8000_bf16", evict("bf16", 16, 8, 128, 16, 3000, 8000, 2000, 500)),
        # one sentence: four beams over an ordinary vocabulary
        ("beam_1x4x32000_fp32", beam("fp32", 1, 4, 32000, 8, 400)),
        # a batch of sentences, some beams ended, over a large vocabulary
        ("beam_32x8x128000_bf16", beam("bf16", 32, 8, 128000, 16, 4000, finished=True)),
    ]
    return [dict(c, name=name) for name, c in named]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def size(lo, hi):
        v = log_int(lo, hi)  # mostly multiples of 8, as models have them
        return max(8, (v + 4) // 8 * 8) if rng.random() < 0.7 else v

    dtype = rng.choice(["fp32", "fp16", "bf16", "bf16"])
    while True:
        op = rng.choice(["linear", "linear", "attend", "attend", "evict", "beam"])
        if op == "linear":
            c = linear(dtype, log_int(1, 4096), size(16, 16384), size(16, 16384), rng.choice(ACTS), rng.random() < 0.6,
                       rng.random() < 0.4, int(rng.random() < 0.7), rng.choice([0, 0, 8, 5]))
            most = 2e10 if dtype == "fp32" else 2.7e11
        elif op == "attend":
            kv = rng.choice([1, 2, 4, 8, 8, 16])
            hi = log_int(1, 131000)
            c = attend(dtype, log_int(1, 64), kv * rng.choice([1, 1, 2, 4, 8, 16, 20]), kv,
                       rng.choice([32, 64, 64, 80, 96, 128, 128, 256, 20, 33]), rng.choice([1, 8, 16, 16, 32, 64, 48, 20]),
                       rng.randint(1, hi), hi, rng.random() < 0.3, rng.random() < 0.4)
            most = 1.1e9
        elif op == "evict":
            hi = log_int(2, 8000)
            budget = rng.randint(1, hi)
            c = evict(dtype, log_int(1, 16), rng.choice([1, 2, 4, 8]), rng.choice([32, 64, 80, 128, 33]),
                      rng.choice([1, 8, 16, 32, 64, 20]), rng.randint(1, hi), hi, budget, rng.randint(0, budget),
                      rng.choice([0, 4]))
            most = 5e8
        else:
            beams = rng.choice([1, 2, 4, 5, 8, 16])
            vocab = log_int(100, 128000)
            c = beam(dtype, log_int(1, 32), beams, vocab, min(beams * rng.choice([1, 2]), vocab), log_int(1, 4000),
                     rng.random() < 0.5)
            most = 7e7
        w = work(c)
        if (w["flops"] if op == "linear" else w["bytes"]) <= most:
            return c


def _lengths(case):
    """Lengths spread evenly over their range: the same work for every seed (which order they come in is the seed's)."""
    s, lo, hi = case["seqs"], case["min_len"], case["max_len"]
    return [hi] if s == 1 else [lo + (hi - lo) * i // (s - 1) for i in range(s)]


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": e * (m * k + n * k + m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)),
                "flops": 2 * m * n * k}
    if case["op"] == "attend":
        total, s, h, kv, d = sum(_lengths(case)), case["seqs"], case["heads"], case["kv_heads"], case["dim"]
        b = 2 * total * kv * d * e + 2 * s * h * d * e + 4 * (total // case["page"] + s) + 4 * s
        b += total if case["mask"] else 0
        b += 8 * total * kv if case["weights"] else 0
        return {"bytes": b, "flops": 4 * total * h * d}
    if case["op"] == "evict":
        b = f = 0
        for n in _lengths(case):
            kept = min(n, case["budget"])
            over = n - kept
            # kept slots behind the budget: the recent ones there, and the heavy ones' share of what is left there
            recent = min(case["recent"], over)
            heavy = max(0, kept - case["recent"] - case["sinks"]) * (over - recent) / max(1, n - case["recent"])
            moved = recent + heavy
            b += case["kv_heads"] * (8 * n + 8 * kept + moved * 4 * case["dim"] * e)
            f += case["kv_heads"] * n
        return {"bytes": int(b), "flops": f}
    rows = case["batch"] * case["beams"]
    return {"bytes": rows * (case["vocab"] * e + 4) + case["batch"] * case["k"] * (12 + 8 * case["state"]),
            "flops": 4 * rows * case["vocab"]}


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _inputs(case, seed):
    """The tensors that a program has in hand before the call."""
    g, t = _gen(seed), TYPES[case["dtype"]]
    if case["op"] == "linear":
        m, n, k, pad = case["m"], case["n"], case["k"], case["pad"]
        st = {"x": _randn(g, m, k + pad, dtype=t)[:, :k]}  # rows of a wider buffer where pad > 0
        st["w"] = (_randn(g, *((n, k) if case["trans_w"] else (k, n))) * k ** -0.5).to(t)
        st["bias"] = (_randn(g, n) * 0.1).to(t) if case["bias"] else None
        st["res"] = _randn(g, m, n, dtype=t) if case["residual"] else None
        st["y"] = torch.empty((m, n), device="cuda", dtype=t)
        return st
    if case["op"] == "beam":
        b, w, v = case["batch"], case["beams"], case["vocab"]
        st = {"logits": (_randn(g, b, w, v) * 2.5).to(t)}
        st["scores"] = -10 * torch.rand((b, w), generator=g, device="cuda")
        st["finished"] = (torch.rand((b, w), generator=g, device="cuda") < 0.25).to(torch.uint8) if case["finished"] else None
        st["end"] = min(2, v - 1)
        st["state"] = torch.randint(0, 1 << 30, (b, w, case["state"]), generator=g, device="cuda", dtype=torch.int32)
        st["next_scores"] = torch.empty((b, case["k"]), device="cuda")
        st["parents"] = torch.empty((b, case["k"]), device="cuda", dtype=torch.int32)
        st["tokens"] = torch.empty((b, case["k"]), device="cuda", dtype=torch.int32)
        st["next_state"] = torch.empty((b, case["k"], case["state"]), device="cuda", dtype=torch.int32)
        return st
    s, kv, d, page = case["seqs"], case["kv_heads"], case["dim"], case["page"]
    pages = -(-case["max_len"] // page)  # of a sequence
    order = torch.randperm(s, generator=g, device="cuda")
    st = {"lengths": torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)[order]}
    st["table"] = torch.randperm(s * pages, generator=g, device="cuda").to(torch.int32).view(s, pages)
    st["k"] = _randn(g, s * pages, kv, page, d, dtype=t)
    st["v"] = _randn(g, s * pages, kv, page, d, dtype=t)
    slots = pages * page
    if case["op"] == "attend":
        h = case["heads"]
        # the query part of a fused projection's rows; scores of a standard deviation of two
        st["qkv"] = _randn(g, s, (h + 2 * kv) * d, dtype=t)
        st["scale"] = 2.0 * d ** -0.5
        st["mask"] = None
        if case["mask"]:  # left-padded prompts: up to a quarter of a sequence's first slots is padding
            first = (torch.rand(s, generator=g, device="cuda") * 0.25 * st["lengths"]).to(torch.int32)
            st["mask"] = (torch.arange(slots, device="cuda") >= first[:, None]).to(torch.uint8)
        st["o"] = torch.empty((s, h, d), device="cuda", dtype=t)
        st["acc"] = st["acc_out"] = None
        if case["weights"]:
            st["acc"] = torch.rand((s, kv, slots), generator=g, device="cuda")
            st["acc_out"] = torch.zeros((s, kv, slots), device="cuda")
        return st
    # weights that a few slots collect most of; positions as tokens came
    st["acc"] = torch.exp(2.0 * _randn(g, s, kv, slots))
    st["pos"] = torch.arange(slots, device="cuda", dtype=torch.int32).expand(s, kv, slots).contiguous()
    st["next"] = st["lengths"].clone()
    st["acc_out"], st["pos_out"] = torch.zeros_like(st["acc"]), torch.zeros_like(st["pos"])
    st["lengths_out"] = torch.zeros_like(st["lengths"])
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if own:
        _plan(st)
    torch.cuda.synchronize()
    return st


def run(st):
    return (_run_own if own else _run_plain)(st)


# ---- through the framework ----

def _plan(st):
    """Descriptors, packed weights and workspaces, as a program keeps them between its calls."""
    from spinn_amd import native as N
    L, c = N.lib(), st["case"]
    N.check(L.spinn_hip_init(0), "spinn_hip_init")
    st["N"], code, p = N, CODES[c["dtype"]], N.ptr

    def workspace(size):
        st["ws"] = torch.empty(size, device="cuda", dtype=torch.uint8) if size else None
        return p(st["ws"]), size

    if c["op"] == "linear":
        act = {"none": N.LINEAR_NONE, "relu": N.LINEAR_RELU, "silu": N.LINEAR_SILU, "gelu": N.LINEAR_GELU,
               "gelu_tanh": N.LINEAR_GELU_TANH}[c["act"]]
        d = N.LinearDesc(m=c["m"], n=c["n"], k=c["k"], dtype=code, trans_w=c["trans_w"], act=act,
                         ldx=st["x"].stride(0), ldres=c["n"], ldy=c["n"])
        st["packed"] = torch.empty(L.spinn_hip_linear_packed_size(C.byref(d)), device="cuda", dtype=torch.uint8)
        N.check(L.spinn_hip_linear_pack_weights(C.byref(d), p(st["w"]), p(st["packed"]), None), "pack")
        ws = workspace(L.spinn_hip_linear_workspace_size(C.byref(d)))
        st["args"] = (C.byref(d), p(st["x"]), p(st["packed"]), p(st["bias"]), p(st["res"]), p(st["y"]), *ws)
        return
    if c["op"] == "beam":
        d = N.BeamDesc(dtype=code, batch=c["batch"], beams=c["beams"], vocab=c["vocab"], k=c["k"], end_token=st["end"],
                       logits_stride=c["vocab"])
        ws = workspace(L.spinn_hip_beam_select_workspace_size(C.byref(d)))
        st["args"] = (C.byref(d), p(st["logits"]), p(st["scores"]), p(st["finished"]), p(st["next_scores"]),
                      p(st["parents"]), p(st["tokens"]), *ws)
        row = 4 * c["state"]
        states = (N.BeamState * 1)(N.BeamState(p(st["state"]), p(st["next_state"]), row, row, row))
        st["reorder"] = (states, 1, c["batch"], c["beams"], c["k"], p(st["parents"]))
        return
    kv, page, dim = c["kv_heads"], c["page"], c["dim"]
    cache = N.KvDesc(dtype=code, seqs=c["seqs"], kv_heads=kv, head_dim=dim, page_size=page, n_pages=st["k"].shape[0],
                     max_pages=st["table"].shape[1], page_stride=kv * page * dim, head_stride=page * dim, slot_stride=dim)
    slots = st["table"].shape[1] * page
    if c["op"] == "attend":
        d = N.KvAttentionDesc(kv=cache, heads=c["heads"], max_len=c["max_len"], scale=st["scale"],
                              q_stride=st["qkv"].stride(0), o_stride=c["heads"] * dim, mask_stride=slots, acc_stride=slots,
                              accumulate=int(c["weights"]))
        ws = workspace(L.spinn_hip_kv_attention_workspace_size(C.byref(d)))
        st["args"] = (C.byref(d), p(st["qkv"]), p(st["k"]), p(st["v"]), p(st["table"]), p(st["lengths"]), p(st["mask"]),
                      p(st["acc"]), p(st["acc_out"]), p(st["o"]), None, *ws)
    else:
        d = N.KvEvictDesc(kv=cache, budget=c["budget"], recent=c["recent"], sinks=c["sinks"], max_len=c["max_len"],
                          acc_stride=slots)
        ws = workspace(L.spinn_hip_kv_evict_workspace_size(C.byref(d)))
        st["args"] = (C.byref(d), p(st["table"]), p(st["lengths"]), p(st["next"]), p(st["acc"]), p(st["pos"]),
                      p(st["acc_out"]), p(st["pos_out"]), p(st["lengths_out"]), p(st["k"]), p(st["v"]), *ws)


def _run_own(st):
    N, op = st["N"], st["case"]["op"]
    L, stream = N.lib(), torch.cuda.current_stream().cuda_stream
    if op == "linear":
        N.check(L.spinn_hip_linear(*st["args"], stream), "spinn_hip_linear")
    elif op == "attend":
        N.check(L.spinn_hip_kv_attention(*st["args"], stream), "spinn_hip_kv_attention")
    elif op == "evict":
        N.check(L.spinn_hip_kv_evict(*st["args"], stream), "spinn_hip_kv_evict")
    else:
        N.check(L.spinn_hip_beam_select(*st["args"], stream), "spinn_hip_beam_select")
        N.check(L.spinn_hip_beam_reorder(*st["reorder"], stream), "spinn_hip_beam_reorder")
    return _outputs(st)


def _outputs(st):
    op = st["case"]["op"]
    if op == "linear":
        return st["y"]
    if op == "attend":
        return {"o": st["o"], **({"acc": st["acc_out"]} if st["acc"] is not None else {})}
    if op == "evict":
        return {"k": st["k"], "v": st["v"], "acc": st["acc_out"], "pos": st["pos_out"], "lengths": st["lengths_out"]}
    return {"scores": st["next_scores"], "parents": st["parents"], "tokens": st["tokens"], "state": st["next_state"]}


# ---- plain forms ----

def _act(v, act):
    if act == "relu":
        return torch.clamp(v, min=0)
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * 2 ** -0.5))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh((2 / math.pi) ** 0.5 * (v + 0.044715 * v * v * v)))
    return v


def _run_plain(st):
    return {"linear": _plain_linear, "attend": _plain_attend, "evict": _plain_evict, "beam": _plain_beam}[st["case"]["op"]](st)


def _plain_linear(st):
    c = st["case"]
    w = st["w"].float()
    v = torch.matmul(st["x"].float(), w.t() if c["trans_w"] else w)
    if c["bias"]:
        v = v + st["bias"].float()
    if c["residual"]:
        v = v + st["res"].float()
    return _act(v, c["act"]).to(st["y"].dtype)


def _rows(pages, table):
    """[seqs, kv heads, slots, dim] in 32 bits of a paged cache."""
    s, n = table.shape
    x = pages[table.reshape(-1).long()].float()
    _, kv, page, d = x.shape
    return x.view(s, n, kv, page, d).transpose(1, 2).reshape(s, kv, n * page, d)


def _plain_attend(st):
    c = st["case"]
    s, h, kv, d = c["seqs"], c["heads"], c["kv_heads"], c["dim"]
    q = st["qkv"][:, :h * d].float().view(s, kv, h // kv, d)
    k, v = _rows(st["k"], st["table"]), _rows(st["v"], st["table"])
    scores = st["scale"] * torch.matmul(k, q.transpose(2, 3).contiguous())  # [seqs, kv heads, slots, group]
    seen = torch.arange(k.shape[2], device=k.device) < st["lengths"][:, None]
    if st["mask"] is not None:
        seen = seen & (st["mask"] != 0)
    seen = seen[:, None, :, None]
    top = torch.where(seen, scores, -math.inf).amax(2, keepdim=True)
    p = torch.where(seen, torch.exp(scores - torch.where(top == -math.inf, 0.0, top)), 0.0)
    total = p.sum(2, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = torch.matmul(p.transpose(2, 3).contiguous(), v).reshape(s, h, d).to(st["o"].dtype)
    if not c["weights"]:
        return {"o": o}
    inside = torch.arange(k.shape[2], device=k.device) < st["lengths"][:, None, None]
    return {"o": o, "acc": torch.where(inside, st["acc"] + p.sum(3), 0.0)}


def _plain_evict(st):
    c = st["case"]
    acc, pos, page = st["acc"], st["pos"], c["page"]
    s, kv, slots = acc.shape
    slot = torch.arange(slots, device=acc.device)
    length = st["lengths"].long()[:, None, None]
    left = torch.clamp(length, max=c["budget"])
    inside = slot < length
    safe = (pos < c["sinks"]) | (pos >= (st["next"][:, None, None] - c["recent"]))
    key = torch.where(inside, torch.where(safe, math.inf, acc), -math.inf)
    rank = torch.sort(key, dim=2, descending=True, stable=True)[1]
    kept = torch.zeros_like(inside.expand(s, kv, slots)).scatter(2, rank, (slot < left).expand(s, kv, slots))
    hole, mover = (slot < left) & ~kept, (slot >= left) & kept
    # the n-th hole takes the n-th kept slot behind the budget
    at = torch.where(mover, mover.long().cumsum(2) - 1, slots)
    movers = torch.zeros((s, kv, slots + 1), device=acc.device, dtype=torch.long).scatter(2, at, slot.expand(s, kv, slots))
    source = torch.where(hole, movers.gather(2, (hole.long().cumsum(2) - 1).clamp(min=0)), slot)
    valid = (slot < left).expand(s, kv, slots)
    acc_out = torch.where(valid, acc.gather(2, source), 0.0)
    pos_out = torch.where(valid, pos.gather(2, source), 0)
    to, source = slot[:c["budget"]].expand(s, kv, -1), source[:, :, :c["budget"]]
    table = st["table"].long()[:, None].expand(s, kv, -1)
    head = torch.arange(kv, device=acc.device)[None, :, None].expand_as(to)
    src_page, dst_page = table.gather(2, source // page), table.gather(2, to // page)
    for t in (st["k"], st["v"]):
        t.index_put_((dst_page, head, to % page), t[src_page, head, source % page])
    return {"k": st["k"], "v": st["v"], "acc": acc_out, "pos": pos_out,
            "lengths": torch.clamp(st["lengths"], max=c["budget"])}


def _plain_beam(st):
    c = st["case"]
    b, w, v, k = c["batch"], c["beams"], c["vocab"], c["k"]
    x = st["logits"].double()
    top = x.amax(2, keepdim=True)
    key = st["scores"].double()[:, :, None] + (x - top - torch.log(torch.exp(x - top).sum(2, keepdim=True)))
    if st["finished"] is not None:  # an ended beam goes on with the end token alone, at its score
        ended = torch.full((v,), -math.inf, device=x.device, dtype=torch.float64)
        ended[st["end"]] = 0.0
        key = torch.where(st["finished"][:, :, None] != 0, st["scores"].double()[:, :, None] + ended, key)
    key = key.view(b, w * v)
    # the k largest; equal ones by the lowest index
    least = torch.topk(key, k, dim=1)[0][:, -1:]
    index = torch.arange(w * v, device=x.device)
    first = torch.topk(torch.where(key == least, -index, -(w * v)), k, dim=1)[0]  # lowest indices at the border
    above = torch.topk(torch.where(key > least, key, -math.inf), k, dim=1)
    at = torch.cat([torch.where(above[0] > -math.inf, above[1], w * v), torch.where(first > -(w * v), -first, w * v)], 1)
    at = torch.sort(at, dim=1)[0]
    val = torch.where(at < w * v, key.gather(1, at.clamp(max=w * v - 1)), -math.inf)
    above_first = torch.where(at < w * v, 0, 1)
    # those above the border come before it; a stable sort by value keeps the lower index first
    order = torch.sort(val, dim=1, descending=True, stable=True)[1]
    order = order.gather(1, torch.sort(above_first.gather(1, order), dim=1, stable=True)[1])[:, :k]
    at = at.gather(1, order)
    parents, tokens = at // v, at % v
    state = st["state"].gather(1, parents[:, :, None].expand(b, k, c["state"]))
    return {"scores": val.gather(1, order).float(), "parents": parents.int(), "tokens": tokens.int(), "state": state}


# ---- what the results are, in 64 bits ----

def exact(case, seed):
    st = _inputs(case, seed)
    if case["op"] == "linear":
        return _exact_linear(case, st)
    if case["op"] == "attend":
        return _exact_attend(case, st)
    if case["op"] == "beam":
        return _exact_beam(case, st)
    return None  # comparisons and copies: nothing is computed


def _exact_linear(case, st):
    w = st["w"].double()
    y = torch.nn.functional.linear(st["x"].double(), w if case["trans_w"] else w.t().contiguous(),
                                   None if st["bias"] is None else st["bias"].double())
    if st["res"] is not None:
        y += st["res"].double()
    if case["act"] == "relu":
        y = torch.relu(y)
    elif case["act"] == "silu":
        y = y * torch.sigmoid(y)
    elif case["act"].startswith("gelu"):
        y = torch.nn.functional.gelu(y, approximate="tanh" if case["act"] == "gelu_tanh" else "none")
    return y


def _exact_attend(case, st):
    """Sequence by sequence, head by head of the cache."""
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    group = h // kv
    o = torch.zeros((case["seqs"], h, d), device="cuda", dtype=torch.float64)
    acc = None if st["acc"] is None else torch.zeros_like(st["acc"], dtype=torch.float64)
    for s, n in enumerate(st["lengths"].tolist()):
        pages = st["table"][s, :-(-n // page)].long()
        for j in range(kv):
            k = st["k"][pages, j].reshape(-1, d)[:n].double()
            v = st["v"][pages, j].reshape(-1, d)[:n].double()
            q = st["qkv"][s, j * group * d:(j + 1) * group * d].view(group, d).double()
            score = torch.mm(q, k.t()) * st["scale"]
            if st["mask"] is not None:
                score = score.masked_fill(st["mask"][s, None, :n] == 0, -math.inf)
            p = torch.softmax(score, 1)
            p = torch.nan_to_num(p, nan=0.0)  # nothing visible
            o[s, j * group:(j + 1) * group] = torch.mm(p, v)
            if acc is not None:
                acc[s, j, :n] = st["acc"][s, j, :n].double() + p.sum(0)
    return {"o": o, **({"acc": acc} if acc is not None else {})}


def _exact_beam(case, st):
    b, w, v, k = case["batch"], case["beams"], case["vocab"], case["k"]
    out = {n: [] for n in ("scores", "parents", "tokens", "state")}
    for i in range(b):
        key = torch.log_softmax(st["logits"][i].double(), -1) + st["scores"][i].double()[:, None]
        if st["finished"] is not None:
            for j in torch.nonzero(st["finished"][i]).flatten().tolist():
                key[j] = -math.inf
                key[j, st["end"]] = st["scores"][i, j].double()
        val, at = torch.sort(key.flatten(), descending=True, stable=True)
        val, at = val[:k], at[:k]
        out["scores"].append(val)
        out["parents"].append(at // v)
        out["tokens"].append(at % v)
        out["state"].append(st["state"][i, at // v])
    return {n: torch.stack(t) for n, t in out.items()}

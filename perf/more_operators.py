"""The operators around a prompt whose speed counts, as plain torch and through the C ABI.

Kinds of case, each a call that a program which generates with this framework makes:

  assign  pages for a step's requests, and where each of their tokens goes, through spinn_hip_kv_assign
  rope    the query and key heads of a fused projection's rows turned by their positions through spinn_hip_rope
  prompt  attention within packed prompts of different lengths through spinn_hip_prompt_attention
  linear8 y = act(x w^T + bias + residual) in 8-bit integers, x quantised row by row within the pass, through
          spinn_hip_quantize_rows and spinn_hip_linear_i8, weights quantised and packed beforehand
"""
import ctypes as C
import math

import torch

own = False  # False: run() computes the plain forms; True: run() calls the framework

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
CODES = {"fp32": 1, "fp16": 10, "bf16": 16}  # ENNF_TYPE_*
ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")


def assign(seqs, page, max_pages, min_new, max_new, prompts, ended, scarce=False):
    return {"op": "assign", "seqs": seqs, "page": page, "max_pages": max_pages, "min_new": min_new, "max_new": max_new,
            "prompts": prompts, "ended": ended, "scarce": scarce}


def rope(dtype, tokens, heads, dim, rot, interleaved, scaling, max_pos, base=10000.0):
    return {"op": "rope", "dtype": dtype, "tokens": tokens, "heads": heads, "dim": dim, "rot": rot,
            "interleaved": interleaved, "scaling": scaling, "max_pos": max_pos, "base": base}


def prompt(dtype, seqs, min_len, max_len, heads, kv_heads, dim, causal=True, before=0, lse=False):
    return {"op": "prompt", "dtype": dtype, "seqs": seqs, "min_len": min_len, "max_len": max_len, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "causal": causal, "before": before, "lse": lse}


def linear8(dtype, m, n, k, act="none", bias=True, residual=False, trans_w=1):
    return {"op": "linear8", "dtype": dtype, "m": m, "n": n, "k": k, "act": act, "bias": bias, "residual": residual,
            "trans_w": trans_w}


def listed():
    named = [
        # a step of generation: every sequence gets one token, one in sixteen a page
        ("assign_64_step", assign(64, 16, 512, 1, 1, 0.0, 0.0)),
        # a busy server's step: some requests end, most generate, some bring prompts
        ("assign_500_mixed", assign(500, 16, 1024, 100, 8000, 0.1, 0.05)),
        # the query and key heads of a batch of single tokens
        ("rope_32x20x128_bf16", rope("bf16", 32, 20, 128, 128, False, "none", 8000)),
        # part of each head in neighbouring pairs, in the graphs' own type
        ("rope_5001x17x80_fp32", rope("fp32", 5001, 17, 80, 32, True, "linear", 20000)),
        # prompts of a batch, context stretched beyond the trained one
        ("rope_16384x40x128_bf16", rope("bf16", 16384, 40, 128, 128, False, "parts", 131072, base=500000.0)),
        # a short question, where latency counts
        ("prompt_1x200_fp16", prompt("fp16", 1, 200, 200, 16, 4, 64)),
        # tokens of images, every one seeing all of its image, heads of their own keys
        ("prompt_8x577_fp32", prompt("fp32", 8, 577, 577, 16, 16, 80, causal=False)),
        # a serving batch of ragged prompts
        ("prompt_24x2000_bf16", prompt("bf16", 24, 37, 2000, 32, 8, 128, lse=True)),
        # one long document
        ("prompt_1x16000_bf16", prompt("bf16", 1, 16000, 16000, 32, 8, 128)),
        # one token through a wide layer: a weight matrix read for a single row
        ("linear8_1x8192x4096_bf16", linear8("bf16", 1, 8192, 4096, "silu", bias=False)),
        # a small batch of sequences back into the residual stream, no multiple of a tile
        ("linear8_45x5120x8192_fp16", linear8("fp16", 45, 5120, 8192, residual=True)),
        # prompts through the wide layer, weights as a MatMul node holds them
        ("linear8_4000x8192x4096_bf16", linear8("bf16", 4000, 8192, 4096, "gelu_tanh", trans_w=0)),
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
        op = rng.choice(["assign", "rope", "prompt", "prompt", "linear8", "linear8"])
        if op == "assign":
            page = rng.choice([1, 8, 16, 16, 20, 32, 64])
            hi = log_int(2, 8000)
            c = assign(log_int(1, 1000), page, max(1, log_int(hi, 32000) // page), rng.randint(1, hi), hi,
                       rng.choice([0.0, 0.1, 0.5, 1.0]), rng.choice([0.0, 0.05, 0.3]), rng.random() < 0.2)
            if c["seqs"] * c["prompts"] * hi <= 1 << 20:
                return c
        elif op == "rope":
            dim = rng.choice([32, 64, 80, 96, 128, 128, 256, 66])
            rot = rng.choice([dim, dim, dim // 2 // 2 * 2, 32])
            c = rope(dtype, log_int(1, 65536), rng.choice([1, 2, 8, 17, 20, 40, 64]), dim, rot, rng.random() < 0.4,
                     rng.choice(["none", "linear", "parts"]), log_int(100, 1000000), rng.choice([10000.0, 500000.0]))
            if work(c)["bytes"] <= 3.4e8:
                return c
        elif op == "prompt":
            kv = rng.choice([1, 2, 4, 8, 8, 16])
            seqs, hi = log_int(1, 64), log_int(1, 16000)
            lo = hi if rng.random() < 0.3 else rng.randint(1, hi)
            before = log_int(1, 4000) if rng.random() < 0.2 else 0
            c = prompt(dtype, seqs, lo, hi, kv * rng.choice([1, 2, 4, 4, 8, 3]), kv, rng.choice([32, 64, 80, 96, 128, 128, 256, 33]),
                       rng.random() < 0.8, before, rng.random() < 0.3)
            scores = seqs * c["heads"] * hi * (hi + before)
            if scores <= 8e9 and work(c)["flops"] <= (1.5e11 if dtype == "fp32" else 1e12):
                return c
        else:
            c = linear8(dtype, log_int(1, 4096), size(16, 16384), size(16, 16384), rng.choice(ACTS), rng.random() < 0.6,
                        rng.random() < 0.4, int(rng.random() < 0.7))
            if work(c)["flops"] <= 2.6e11:
                return c


def _spread(s, lo, hi):
    """Lengths spread evenly over their range: the same work for every seed (which order they come in is the seed's)."""
    return [hi] if s == 1 else [lo + (hi - lo) * i // (s - 1) for i in range(s)]


def _requests(case):
    """How many sequences bring prompts of which lengths, how many end; the others get one token."""
    ended = int(case["seqs"] * case["ended"])
    prompts = min(int(round(case["seqs"] * case["prompts"])), case["seqs"] - ended)
    capacity = case["page"] * case["max_pages"]
    return [min(n, capacity) for n in _spread(prompts, case["min_new"], case["max_new"])] if prompts else [], ended


def _inverse(case):
    """Angle per position of each pair, in 64 bits."""
    i = torch.arange(case["rot"] // 2, dtype=torch.float64, device="cuda")
    f = torch.exp(-2.0 * i / case["rot"] * math.log(case["base"]))
    if case["scaling"] == "linear":
        f = f / 4.0
    elif case["scaling"] == "parts":  # pairs that turn 4 times or more within 8192 positions stay, those under one are stretched
        turns = 8192 * f / (2 * math.pi)
        stay = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = stay * f + (1 - stay) * f / 8.0
    return f


def work(case):
    if case["op"] == "assign":
        prompts, ended = _requests(case)
        tokens = sum(prompts) + case["seqs"] - len(prompts) - ended
        return {"bytes": 40 * case["seqs"] + 12 * tokens + 8 * (tokens // case["page"]), "flops": 4 * tokens}
    e = BYTES[case["dtype"]]
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * e * n + 4 * case["tokens"] + 8 * (case["rot"] // 2),
                "flops": 3 * case["tokens"] * case["heads"] * case["rot"]}
    if case["op"] == "prompt":
        h, kv, d, b = case["heads"], case["kv_heads"], case["dim"], case["before"]
        lens = _spread(case["seqs"], case["min_len"], case["max_len"])
        pairs = sum(n * (b + n) - (n * (n - 1) // 2 if case["causal"] else 0) for n in lens)
        rows = sum(lens)
        return {"bytes": e * d * (2 * rows * h + 2 * (rows + len(lens) * b) * kv) + (4 * rows * h if case["lse"] else 0),
                "flops": 4 * pairs * h * d}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": e * (m * k + m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)) + n * k + 4 * (n + m),
            "flops": 2 * m * n * k}


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _inputs(case, seed):
    """The tensors that a program has in hand before the call."""
    return {"assign": _assign_inputs, "rope": _rope_inputs, "prompt": _prompt_inputs, "linear8": _linear8_inputs}[case["op"]](case, _gen(seed))


def _i32(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _starts(lens):
    return torch.cat([torch.zeros_like(lens[:1]), torch.cumsum(lens, 0, dtype=torch.int32)])


def _assign_inputs(c, g):
    s, page, row = c["seqs"], c["page"], c["max_pages"]
    prompts, ended = _requests(c)
    order = torch.randperm(s, generator=g, device="cuda")
    new = _i32(prompts + [-1] * ended + [1] * (s - len(prompts) - ended))[order]
    # those that go on have up to a row but a token, those that begin nothing
    lengths = (torch.rand(s, generator=g, device="cuda") * (page * row - 1)).to(torch.int32).clamp(min=0)
    lengths = torch.where(order < len(prompts), 0, lengths)
    held = (lengths + page - 1) // page
    # pages in random places: the sequences' own first, then the free ones (with scarce: half of what could be asked for)
    free = sum(-(-n // page) for n in prompts) + s
    free = max(1, free // 2) if c["scarce"] else free
    total = s * row + free
    pages = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    st = {"new": new, "lengths": lengths, "held": held, "next": lengths.clone(), "table": pages[:s * row].view(s, row).contiguous()}
    st["free"] = torch.full((total,), -1, device="cuda", dtype=torch.int32)
    st["free"][:free] = pages[s * row:]
    st["free_count"] = _i32([free])
    st["max_tokens"] = (sum(prompts) + s - len(prompts) - ended + 63) // 64 * 64
    st["pages"] = total
    for n in ("lengths", "held", "next", "free_count"):
        st[n + "_out"] = torch.zeros_like(st[n])
    st["starts"], st["served"] = torch.zeros(s + 1, device="cuda", dtype=torch.int32), torch.zeros(s, device="cuda", dtype=torch.int32)
    for n in ("seq", "slot", "position"):
        st[n] = torch.zeros(st["max_tokens"], device="cuda", dtype=torch.int32)
    return st


def _rope_inputs(c, g):
    t = TYPES[c["dtype"]]
    width = (c["heads"] + max(1, c["heads"] // 5)) * c["dim"]  # values follow the query and key heads in a projection's rows
    st = {"x": _randn(g, c["tokens"], width, dtype=t)}
    st["position"] = torch.randint(0, c["max_pos"], (c["tokens"],), generator=g, device="cuda", dtype=torch.int32)
    st["y"] = torch.empty((c["tokens"], c["heads"], c["dim"]), device="cuda", dtype=t)
    return st


def _prompt_inputs(c, g):
    t, h, kv, d = TYPES[c["dtype"]], c["heads"], c["kv_heads"], c["dim"]
    order = torch.randperm(c["seqs"], generator=g, device="cuda")
    lens = _i32(_spread(c["seqs"], c["min_len"], c["max_len"]))[order]
    rows = sum(_spread(c["seqs"], c["min_len"], c["max_len"]))
    st = {"starts": _starts(lens), "kv_starts": None}
    # a fused projection's rows; with keys of its own before each prompt, these are in arrays of their own
    st["qkv"] = _randn(g, rows, (h + 2 * kv) * d, dtype=t)
    st["q"] = st["qkv"][:, :h * d]
    st["k"], st["v"] = st["qkv"][:, h * d:(h + kv) * d], st["qkv"][:, (h + kv) * d:]
    if c["before"]:
        st["kv_starts"] = _starts(lens + c["before"])
        st["k"], st["v"] = (_randn(g, rows + c["seqs"] * c["before"], kv * d, dtype=t) for _ in range(2))
    st["scale"] = 2.0 * d ** -0.5  # scores of a standard deviation of two
    st["o"] = torch.empty((rows, h, d), device="cuda", dtype=t)
    st["lse"] = torch.empty((rows, h), device="cuda") if c["lse"] else None
    return st


def _linear8_inputs(c, g):
    t, m, n, k = TYPES[c["dtype"]], c["m"], c["n"], c["k"]
    st = {"x": _randn(g, m, k, dtype=t)}
    # weights of unit variance over k, their channels' scales from the largest of each
    st["wq"] = torch.randint(-127, 128, (n, k) if c["trans_w"] else (k, n), generator=g, device="cuda", dtype=torch.int8)
    st["ws"] = (0.75 + 0.5 * torch.rand(n, generator=g, device="cuda")) * (k ** -0.5 / 73.0)
    st["bias"] = (_randn(g, n) * 0.1).to(t) if c["bias"] else None
    st["res"] = _randn(g, m, n, dtype=t) if c["residual"] else None
    st["xq"] = torch.empty((m, (k + 15) // 16 * 16), device="cuda", dtype=torch.int8)
    st["xs"] = torch.empty(m, device="cuda")
    st["y"] = torch.empty((m, n), device="cuda", dtype=t)
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if own:
        _plan(st)
    else:
        _plain_plan(st)
    torch.cuda.synchronize()
    return st


def run(st):
    return (_run_own if own else _run_plain)(st)


# ---- through the framework ----

def _plan(st):
    """Descriptors, packed weights, tables and workspaces, as a program keeps them between its calls."""
    from spinn_amd import native as N
    L, c = N.lib(), st["case"]
    N.check(L.spinn_hip_init(0), "spinn_hip_init")
    st["N"], p = N, N.ptr

    def workspace(size):
        st["space"] = torch.empty(size, device="cuda", dtype=torch.uint8) if size else None
        return p(st["space"]), size

    if c["op"] == "assign":
        d = N.KvAssignDesc(seqs=c["seqs"], page_size=c["page"], n_pages=st["pages"], max_pages=c["max_pages"],
                           max_tokens=st["max_tokens"])
        st["calls"] = [("spinn_hip_kv_assign", (C.byref(d), *(p(st[n]) for n in (
            "new", "lengths", "next", "held", "free_count", "free", "table", "lengths_out", "next_out", "held_out",
            "free_count_out", "starts", "served", "seq", "slot", "position"))))]
        return
    code = CODES[c["dtype"]]
    if c["op"] == "rope":
        kinds = {"none": N.ROPE_PLAIN, "linear": N.ROPE_LINEAR, "parts": N.ROPE_BY_PARTS}
        d = N.RopeDesc(dtype=code, heads=c["heads"], head_dim=c["dim"], rot_dim=c["rot"], interleaved=int(c["interleaved"]),
                       scaling=kinds[c["scaling"]], base=c["base"], factor={"none": 1.0, "linear": 4.0, "parts": 8.0}[c["scaling"]],
                       low=1.0, high=4.0, trained=8192, magnitude=1.0, x_stride=st["x"].stride(0), x_head_stride=c["dim"],
                       y_stride=c["heads"] * c["dim"], y_head_stride=c["dim"])
        st["turns"] = torch.empty(L.spinn_hip_rope_table_size(C.byref(d)), device="cuda", dtype=torch.uint8)
        N.check(L.spinn_hip_rope_table(C.byref(d), p(st["turns"]), None), "table")
        st["calls"] = [("spinn_hip_rope", (C.byref(d), c["tokens"], p(st["position"]), p(st["turns"]), p(st["x"]), p(st["y"])))]
    elif c["op"] == "prompt":
        h, kv, dim = c["heads"], c["kv_heads"], c["dim"]
        d = N.PromptAttentionDesc(dtype=code, seqs=c["seqs"], heads=h, kv_heads=kv, head_dim=dim, causal=int(c["causal"]),
                                  q_rows=st["q"].shape[0], kv_rows=st["k"].shape[0], scale=st["scale"], q_stride=st["q"].stride(0),
                                  k_stride=st["k"].stride(0), v_stride=st["v"].stride(0), o_stride=h * dim)
        space = workspace(L.spinn_hip_prompt_attention_workspace_size(C.byref(d)))
        st["calls"] = [("spinn_hip_prompt_attention", (C.byref(d), p(st["q"]), p(st["k"]), p(st["v"]), p(st["starts"]),
                                                       p(st["kv_starts"]), p(st["o"]), p(st["lse"]), *space))]
    else:
        act = {"none": N.LINEAR_NONE, "relu": N.LINEAR_RELU, "silu": N.LINEAR_SILU, "gelu": N.LINEAR_GELU,
               "gelu_tanh": N.LINEAR_GELU_TANH}[c["act"]]
        d = N.LinearI8Desc(m=c["m"], n=c["n"], k=c["k"], dtype=code, trans_w=c["trans_w"], act=act, ldx=st["xq"].stride(0),
                           ldres=c["n"], ldy=c["n"])
        st["packed"] = torch.empty(L.spinn_hip_linear_i8_packed_size(C.byref(d)), device="cuda", dtype=torch.uint8)
        N.check(L.spinn_hip_linear_i8_pack_weights(C.byref(d), p(st["wq"]), p(st["packed"]), None), "pack")
        space = workspace(L.spinn_hip_linear_i8_workspace_size(C.byref(d)))
        st["calls"] = [("spinn_hip_quantize_rows", (code, c["m"], c["k"], p(st["x"]), c["k"], p(st["xq"]), st["xq"].stride(0), p(st["xs"]))),
                       ("spinn_hip_linear_i8", (C.byref(d), p(st["xq"]), p(st["xs"]), p(st["packed"]), p(st["ws"]), p(st["bias"]),
                                                p(st["res"]), p(st["y"]), *space))]


def _run_own(st):
    N = st["N"]
    L, stream = N.lib(), torch.cuda.current_stream().cuda_stream
    for name, args in st["calls"]:
        N.check(getattr(L, name)(*args, stream), name)
    return _outputs(st)


def _outputs(st):
    op = st["case"]["op"]
    if op == "assign":
        return {n: st[n] for n in ("lengths_out", "next_out", "held_out", "free_count_out", "starts", "served", "seq", "slot",
                                   "position", "table", "free")}
    if op == "rope":
        return st["y"]
    if op == "prompt":
        return {"o": st["o"], **({"lse": st["lse"]} if st["lse"] is not None else {})}
    return {"y": st["y"], "scale": st["xs"]}


# ---- plain forms ----

def _plain_plan(st):
    """What a program of plain torch would keep: weights in 64 bits (integer products pass 24 bits), frequencies, the longest lengths."""
    c = st["case"]
    if c["op"] == "linear8":
        w = st["wq"].double()
        st["wide"] = w.t().contiguous() if c["trans_w"] else w
    elif c["op"] == "rope":
        st["inverse"] = _inverse(c)


def _run_plain(st):
    return {"assign": _plain_assign, "rope": _plain_rope, "prompt": _plain_prompt, "linear8": _plain_linear8}[st["case"]["op"]](st)


def _plain_assign(st):
    c = st["case"]
    page, row, s = c["page"], c["max_pages"], c["seqs"]
    new, length, held, table, free = (st[n].long() for n in ("new", "lengths", "held", "table", "free"))
    ended, add = new == -1, new.clamp(min=0)
    ends = add.cumsum(0)
    starts = (ends - add).clamp(max=st["max_tokens"])
    fits = (new >= -1) & ((add == 0) | (length + add <= page * row) & (ends <= st["max_tokens"]))
    # pages of ended sequences go on top of the free ones, in the sequences' order
    back = torch.where(ended, held, 0)
    place = st["free_count"].long() + back.cumsum(0) - back
    col = torch.arange(row, device="cuda")
    gives = ended[:, None] & (col < held[:, None])
    seat = torch.where(gives, place[:, None] + col, free.numel())
    free = torch.cat([free, free[:1]]).scatter(0, seat.flatten(), torch.where(gives, table, 0).flatten())[:-1]
    count = st["free_count"].long() + back.sum()
    need = torch.where(fits & (add > 0), ((length + add + page - 1) // page - held).clamp(min=0), 0)
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= count))
    got = torch.where(served, need, 0)
    # page j of a sequence's new ones is number (those before it) + j from the top
    takes = (col >= held[:, None]) & (col < (held + got)[:, None])
    source = count - 1 - ((upto - need)[:, None] + col - held[:, None])
    table = torch.where(takes, free[source.clamp(0, free.numel() - 1)], table)
    taken = got.sum()
    token = torch.arange(st["max_tokens"], device="cuda")
    owner = (torch.searchsorted(ends, token, right=True)).clamp(max=s - 1)
    real = (token < ends[-1]) & served[owner]
    at = token - starts[owner]
    grown = torch.where(served, add, 0)
    out = {"lengths_out": torch.where(ended, 0, length + grown), "next_out": torch.where(ended, 0, st["next"].long() + grown),
           "held_out": torch.where(ended, 0, held + got), "free_count_out": (count - taken).view(1),
           "starts": torch.cat([starts, ends[-1:].clamp(max=st["max_tokens"])]), "served": served,
           "seq": torch.where(real, owner, -1), "slot": torch.where(real, length[owner] + at, -1),
           "position": torch.where(real, st["next"].long()[owner] + at, 0), "table": table, "free": free}
    return {n: t.to(torch.int32) for n, t in out.items()}


def _plain_rope(st):
    c = st["case"]
    rot, half = c["rot"], c["rot"] // 2
    x = st["x"][:, :c["heads"] * c["dim"]].reshape(c["tokens"], c["heads"], c["dim"]).float()
    angle = st["position"].double()[:, None] * st["inverse"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if c["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(2)
    else:
        a, b = x[..., :half], x[..., half:rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, x[..., rot:]], -1).to(st["y"].dtype)


def _plain_prompt(st):
    """Every sequence in a padded batch."""
    c = st["case"]
    s, h, kv, d = c["seqs"], c["heads"], c["kv_heads"], c["dim"]
    starts = st["starts"].long()
    kv_starts = starts if st["kv_starts"] is None else st["kv_starts"].long()
    i, j = (torch.arange(n, device="cuda") for n in (c["max_len"], c["max_len"] + c["before"]))
    nq, nk = starts[1:] - starts[:-1], kv_starts[1:] - kv_starts[:-1]
    row = (starts[:-1, None] + i).clamp(max=st["q"].shape[0] - 1)
    col = (kv_starts[:-1, None] + j).clamp(max=st["k"].shape[0] - 1)
    q = st["q"][row].float().view(s, i.numel(), kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(s, kv, -1, d)
    k = st["k"][col].float().view(s, j.numel(), kv, d).permute(0, 2, 3, 1).contiguous()
    v = st["v"][col].float().view(s, j.numel(), kv, d).transpose(1, 2).contiguous()
    scores = torch.matmul(q, k).mul_(st["scale"]).view(s, kv, h // kv, i.numel(), j.numel())
    seen = (j < nk[:, None])[:, None]
    if c["causal"]:
        seen = seen & (j <= i[:, None] + (nk - nq)[:, None, None])
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(s, kv, -1, j.numel()), v).view(s, kv, h // kv, i.numel(), d)
    o = o / torch.where(total == 0, 1.0, total)
    inside = i < nq[:, None]
    out = {"o": o.permute(0, 3, 1, 2, 4).reshape(s, i.numel(), h, d)[inside].to(st["o"].dtype)}
    if st["lse"] is not None:
        lse = (top + torch.log(total)).squeeze(-1)
        out["lse"] = lse.permute(0, 3, 1, 2).reshape(s, i.numel(), h)[inside]
    return out


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


def _plain_linear8(st):
    c = st["case"]
    x = st["x"].float()
    scale = (x.abs().amax(1).double() / 127).float()
    xq = torch.round(x.double() / torch.where(scale == 0, 1.0, scale).double()[:, None]).clamp(-127, 127)  # next to a border in 64 bits
    v = torch.matmul(xq, st["wide"]).float() * scale[:, None] * st["ws"]
    if c["bias"]:
        v = v + st["bias"].float()
    if c["residual"]:
        v = v + st["res"].float()
    return {"y": _act(v, c["act"]).to(st["y"].dtype), "scale": scale}


# ---- what the results are, in 64 bits ----

def exact(case, seed):
    if case["op"] == "assign":
        return None  # counts and copies: nothing is computed
    st = _inputs(case, seed)
    return {"rope": _exact_rope, "prompt": _exact_prompt, "linear8": _exact_linear8}[case["op"]](case, st)


def _exact_rope(c, st):
    """Each pair as a complex number."""
    x = st["x"][:, :c["heads"] * c["dim"]].double().reshape(c["tokens"], c["heads"], c["dim"])
    turned, rest = x[..., :c["rot"]], x[..., c["rot"]:]
    pairs = turned.unflatten(2, (-1, 2)) if c["interleaved"] else turned.unflatten(2, (2, -1)).transpose(2, 3)
    z = torch.view_as_complex(pairs.contiguous())
    angle = torch.outer(st["position"].double(), _inverse(c))
    pairs = torch.view_as_real(z * torch.polar(torch.ones_like(angle), angle)[:, None])
    turned = pairs.flatten(2) if c["interleaved"] else pairs.transpose(2, 3).flatten(2)
    return torch.cat([turned, rest], 2)


def _exact_prompt(c, st):
    """Sequence by sequence, head by head, in blocks of rows."""
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    rows = st["q"].shape[0]
    o = torch.zeros((rows, h, d), device="cuda", dtype=torch.float64)
    lse = torch.full((rows, h), -math.inf, device="cuda", dtype=torch.float64)
    starts = st["starts"].tolist()
    kv_starts = starts if st["kv_starts"] is None else st["kv_starts"].tolist()
    for q0, q1, k0, k1 in zip(starts, starts[1:], kv_starts, kv_starts[1:]):
        for x in range(h):
            g = x // (h // kv)
            k, v = st["k"][k0:k1, g * d:(g + 1) * d].double(), st["v"][k0:k1, g * d:(g + 1) * d].double()
            kt = k.t().contiguous()
            for a in range(q0, q1, 4096):
                b = min(q1, a + 4096)
                score = torch.mm(st["q"][a:b, x * d:(x + 1) * d].double(), kt) * st["scale"]
                if c["causal"]:
                    last = torch.arange(a - q0, b - q0, device="cuda") + (k1 - k0) - (q1 - q0)
                    score.masked_fill_(torch.arange(k1 - k0, device="cuda") > last[:, None], -math.inf)
                lse[a:b, x] = torch.logsumexp(score, 1)
                o[a:b, x] = torch.mm(torch.softmax(score, 1), v)
    return {"o": o, **({"lse": lse} if c["lse"] else {})}


def _exact_linear8(c, st):
    x = st["x"].double()
    scale = (x.abs().max(1).values / 127).float()  # held in 32 bits by definition
    s = scale.double()
    q = torch.where(s[:, None] > 0, x / s[:, None], 0.0).round().clamp(-127, 127)
    w = st["wq"].double() if c["trans_w"] else st["wq"].double().t().contiguous()
    y = torch.nn.functional.linear(q, w) * torch.outer(s, st["ws"].double())
    if st["bias"] is not None:
        y += st["bias"].double()
    if st["res"] is not None:
        y += st["res"].double()
    if c["act"] == "relu":
        y = torch.relu(y)
    elif c["act"] == "silu":
        y = y * torch.sigmoid(y)
    elif c["act"].startswith("gelu"):
        y = torch.nn.functional.gelu(y, approximate="tanh" if c["act"] == "gelu_tanh" else "none")
    return {"y": y, "scale": scale}

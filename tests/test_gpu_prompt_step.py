"""The operators around a prompt and those of a decoding step together, as a server runs them: requests come and go,
pages and slots are assigned on the device, projections run in 8-bit integers, positions are turned, keys and values
go into the paged cache, prompts attend within themselves and single tokens over the cache."""
import ctypes as C

import pytest
import torch

from tests.decodeops import BF16, F32, TORCH, gen, ptr, randn, stream, workspace

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, WIDTH, PAGE, ROW, PAGES = 8, 2, 64, 256, 16, 12, 64
SLOTS = PAGE * ROW


class Server:
    """One attention layer over a paged cache; everything between the calls stays on the device."""

    def __init__(self, N, dtype, seqs, max_tokens):
        self.N, self.L, self.dtype, self.seqs, self.max_tokens = N, N.lib(), dtype, seqs, max_tokens
        g = gen(1)
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
        t = TORCH[dtype]
        self.new, self.lengths, self.next, self.held = i32(seqs), i32(seqs), i32(seqs), i32(seqs)
        self.table = torch.full((seqs, ROW), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(PAGES, generator=g).to(torch.int32).cuda()
        self.count = torch.tensor([PAGES], dtype=torch.int32, device="cuda")
        self.starts, self.served = i32(seqs + 1), i32(seqs)
        self.seq, self.slot, self.position = i32(max_tokens), i32(max_tokens), i32(max_tokens)
        self.k = torch.full((PAGES, KV, PAGE, DIM), float("nan"), dtype=t, device="cuda")
        self.v = self.k.clone()
        self.x = torch.zeros((max_tokens, WIDTH), dtype=t, device="cuda")
        self.n = (HEADS + 2 * KV) * DIM
        self.rows = torch.zeros((max_tokens, self.n), dtype=t, device="cuda")
        self.o = torch.zeros((max_tokens, HEADS * DIM), dtype=t, device="cuda")
        self.xq, self.xs = torch.zeros((max_tokens, WIDTH), dtype=torch.int8, device="cuda"), torch.zeros(max_tokens, device="cuda")
        w = randn(g, self.n, WIDTH, scale=WIDTH ** -0.5).cuda()
        self.wq, self.ws = torch.zeros((self.n, WIDTH), dtype=torch.int8, device="cuda"), torch.zeros(self.n, device="cuda")
        N.check(self.L.spinn_hip_quantize_rows(F32, self.n, WIDTH, ptr(w), WIDTH, ptr(self.wq), WIDTH, ptr(self.ws), stream()), "weights")
        d = self.linear_desc(1)
        self.packed = torch.zeros(self.L.spinn_hip_linear_i8_packed_size(C.byref(d)), dtype=torch.uint8, device="cuda")
        N.check(self.L.spinn_hip_linear_i8_pack_weights(C.byref(d), ptr(self.wq), ptr(self.packed), stream()), "pack")
        self.rope = N.RopeDesc(dtype=dtype, heads=HEADS + KV, head_dim=DIM, rot_dim=DIM, interleaved=0, scaling=1, base=10000.0, factor=2.0,
                               magnitude=1.0, x_stride=self.n, x_head_stride=DIM, y_stride=self.n, y_head_stride=DIM)
        self.turns = torch.zeros(self.L.spinn_hip_rope_table_size(C.byref(self.rope)), dtype=torch.uint8, device="cuda")
        N.check(self.L.spinn_hip_rope_table(C.byref(self.rope), ptr(self.turns), stream()), "table")
        self.kv = N.KvDesc(dtype=dtype, seqs=seqs, kv_heads=KV, head_dim=DIM, page_size=PAGE, n_pages=PAGES, max_pages=ROW,
                           page_stride=KV * PAGE * DIM, head_stride=PAGE * DIM, slot_stride=DIM)
        self.spaces = {}

    def linear_desc(self, m):
        return self.N.LinearI8Desc(m=m, n=self.n, k=WIDTH, dtype=self.dtype, trans_w=1)

    def space(self, name, size):
        if name not in self.spaces:
            self.spaces[name] = workspace(size)
        return ptr(self.spaces[name]), size

    def before_attention(self, tokens):
        """Pages, projections, positions and the cache for the first `tokens` rows of x."""
        N, L = self.N, self.L
        a = N.KvAssignDesc(seqs=self.seqs, page_size=PAGE, n_pages=PAGES, max_pages=ROW, max_tokens=tokens)
        N.check(L.spinn_hip_kv_assign(C.byref(a), ptr(self.new), ptr(self.lengths), ptr(self.next), ptr(self.held), ptr(self.count), ptr(self.free),
                                      ptr(self.table), ptr(self.lengths), ptr(self.next), ptr(self.held), ptr(self.count), ptr(self.starts),
                                      ptr(self.served), ptr(self.seq), ptr(self.slot), ptr(self.position), stream()), "assign")
        d = self.linear_desc(tokens)
        N.check(L.spinn_hip_quantize_rows(self.dtype, tokens, WIDTH, ptr(self.x), WIDTH, ptr(self.xq), WIDTH, ptr(self.xs), stream()), "quantize")
        N.check(L.spinn_hip_linear_i8(C.byref(d), ptr(self.xq), ptr(self.xs), ptr(self.packed), ptr(self.ws), None, None, ptr(self.rows),
                                      *self.space(("linear", tokens), L.spinn_hip_linear_i8_workspace_size(C.byref(d))), stream()), "linear")
        N.check(L.spinn_hip_rope(C.byref(self.rope), tokens, ptr(self.position), ptr(self.turns), ptr(self.rows), ptr(self.rows), stream()), "rope")
        self.parts = (self.rows[:, :HEADS * DIM], self.rows[:, HEADS * DIM:(HEADS + KV) * DIM], self.rows[:, (HEADS + KV) * DIM:])
        _, k, v = self.parts
        N.check(L.spinn_hip_kv_append(C.byref(self.kv), tokens, ptr(self.seq), ptr(self.slot), ptr(self.position), ptr(k), self.n, ptr(v), self.n,
                                      ptr(self.table), ptr(self.k), ptr(self.v), None, None, 0, stream()), "append")

    def prompts(self, tokens):
        self.before_attention(tokens)
        q, k, v = self.parts
        d = self.N.PromptAttentionDesc(dtype=self.dtype, seqs=self.seqs, heads=HEADS, kv_heads=KV, head_dim=DIM, causal=1, q_rows=tokens,
                                       kv_rows=tokens, scale=DIM ** -0.5, q_stride=self.n, k_stride=self.n, v_stride=self.n, o_stride=HEADS * DIM)
        self.N.check(self.L.spinn_hip_prompt_attention(
            C.byref(d), ptr(q), ptr(k), ptr(v), ptr(self.starts), None, ptr(self.o), None,
            *self.space(("prompt", tokens), self.L.spinn_hip_prompt_attention_workspace_size(C.byref(d))), stream()), "prompt")

    def tokens(self):
        """One token of every sequence: row s of x is sequence s's."""
        self.before_attention(self.seqs)
        d = self.N.KvAttentionDesc(kv=self.kv, heads=HEADS, max_len=SLOTS, scale=DIM ** -0.5, q_stride=self.n, o_stride=HEADS * DIM)
        self.N.check(self.L.spinn_hip_kv_attention(
            C.byref(d), ptr(self.parts[0]), ptr(self.k), ptr(self.v), ptr(self.table), ptr(self.lengths), None, None, None, ptr(self.o), None,
            *self.space("attend", self.L.spinn_hip_kv_attention_workspace_size(C.byref(d))), stream()), "attend")


def close(got, want, what):
    """Both attentions are within a rounding of the result's type of the exact one, and the weights' roundings before (bf16: 2^-8 each)."""
    tol = 3 * 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -17
    d = (got.double() - want.double()).abs().max().item()
    bound = tol * want.double().abs().max().item()
    print(f"[bound] {what}: {d / bound:.3f} of the bound", flush=True)
    assert d <= bound, what


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_prompt_at_once_and_token_by_token(hip, dtype):
    """A prompt through the prompt's attention leaves the cache and the results that its tokens one by one do."""
    lens = [37, 5, 90, 1]
    total = sum(lens)
    at_once, one_by_one = Server(hip, dtype, 4, total), Server(hip, dtype, 4, total)
    at_once.x.copy_(randn(gen(2), total, WIDTH, dtype=dtype))
    at_once.new.copy_(torch.tensor(lens, dtype=torch.int32))
    at_once.prompts(total)
    assert at_once.served.tolist() == [1] * 4 and at_once.lengths.tolist() == lens and at_once.starts.tolist() == [0, 37, 42, 132, 133]
    first = at_once.starts[:-1].tolist()
    for i in range(max(lens)):
        new = [int(i < n) for n in lens]
        one_by_one.new.copy_(torch.tensor(new, dtype=torch.int32))
        # tokens are packed: rows of the sequences that still have one
        live = [s for s in range(4) if new[s]]
        one_by_one.x[:len(live)] = at_once.x[[first[s] + i for s in live]]
        one_by_one.before_attention(4)
        d = hip.KvAttentionDesc(kv=one_by_one.kv, heads=HEADS, max_len=SLOTS, scale=DIM ** -0.5, q_stride=one_by_one.n, o_stride=HEADS * DIM)
        q = torch.zeros((4, one_by_one.n), dtype=TORCH[dtype], device="cuda")
        q[live] = one_by_one.rows[:len(live)]
        o = torch.zeros((4, HEADS * DIM), dtype=TORCH[dtype], device="cuda")
        hip.check(hip.lib().spinn_hip_kv_attention(
            C.byref(d), ptr(q), ptr(one_by_one.k), ptr(one_by_one.v), ptr(one_by_one.table), ptr(one_by_one.lengths), None, None, None, ptr(o), None,
            *one_by_one.space("attend", hip.lib().spinn_hip_kv_attention_workspace_size(C.byref(d))), stream()), "attend")
        for s in live:
            close(o[s], at_once.o[first[s] + i], f"token {i} of {s}")
    assert one_by_one.lengths.tolist() == lens

    def cached(srv, s, t):
        return t[srv.table[s, :-(-lens[s] // PAGE)].long()].transpose(0, 1).reshape(KV, -1, DIM)[:, :lens[s]]

    for s in range(4):
        for a, b in ((at_once.k, one_by_one.k), (at_once.v, one_by_one.v)):
            assert torch.equal(cached(at_once, s, a), cached(one_by_one, s, b))


def test_requests_come_and_go(hip):
    """Prompts, then captured steps of single tokens, an end, a new prompt in the freed pages, more steps: every result against plain torch
    in 64 bits on the rows that the projections gave."""
    srv = Server(hip, BF16, 3, 160)
    g = gen(3)
    history = {}  # sequence: list of (k, v) rows

    def follow(rows_of):
        """Exact results of the rows (sequence s: its rows of srv.rows)."""
        torch.cuda.synchronize()
        for s, rows in rows_of.items():
            for i, r in enumerate(rows):
                row = srv.rows[r].double().cpu()
                k, v = row[HEADS * DIM:(HEADS + KV) * DIM].view(KV, DIM), row[(HEADS + KV) * DIM:].view(KV, DIM)
                history.setdefault(s, []).append((k, v))
                ks, vs = torch.stack([a for a, _ in history[s]], 1), torch.stack([b for _, b in history[s]], 1)
                q = row[:HEADS * DIM].view(KV, HEADS // KV, DIM)
                p = torch.softmax((q @ ks.transpose(1, 2)) * DIM ** -0.5, -1)
                close(srv.o[r].cpu(), (p @ vs).reshape(-1), f"sequence {s}, token {len(history[s])}")
                assert int(srv.position[r]) == len(history[s]) - 1

    def prompts(lens):
        srv.new.copy_(torch.tensor(lens, dtype=torch.int32))
        srv.x.copy_(randn(g, 160, WIDTH, dtype=BF16))
        srv.prompts(160)
        start, rows = 0, {}
        for s, n in enumerate(lens):
            if n > 0:
                rows[s] = range(start, start + n)
                start += n
            elif n < 0:
                history.pop(s, None)
        follow(rows)

    prompts([40, 17, 90])
    graph = torch.cuda.CUDAGraph()
    srv.new.fill_(1)
    with torch.cuda.graph(graph):
        srv.tokens()

    def steps(n):
        for _ in range(n):
            srv.new.fill_(1)
            srv.x[:3] = randn(g, 3, WIDTH, dtype=BF16).cuda()
            graph.replay()
            follow({s: [s] for s in range(3)})

    steps(9)
    used = PAGES - int(srv.count)
    assert used == sum(-(-n // PAGE) for n in (49, 26, 99))
    prompts([-1, 0, 0])
    assert srv.lengths.tolist() == [0, 26, 99] and int(srv.count) == PAGES - 2 - 7
    prompts([120, 0, 0])
    steps(8)
    assert srv.lengths.tolist() == [128, 34, 107]
    assert srv.table[0, :8].tolist() != [-1] * 8
    held = [srv.table[s, :int(srv.held[s])].tolist() for s in range(3)]
    names = sum(held, [])
    assert len(set(names)) == len(names), "a page given twice"
    assert set(names).isdisjoint(srv.free[:int(srv.count)].tolist())

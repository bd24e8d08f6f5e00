"""A server's steps that mix prompts, single tokens, idle and ended requests, without a look at the device's data: pages are assigned to the prompts,
then to the single tokens; these rows' queries go to their sequences' rows and the results back by spinn_hip_beam_reorder."""
import ctypes as C

import pytest
import torch

from tests.decodeops import BF16, F32, gen, ptr, randn, stream
from tests.test_gpu_prompt_step import DIM, HEADS, KV, PAGE, PAGES, ROW, SLOTS, WIDTH, Server, close

pytestmark = pytest.mark.gpu


class Mixed(Server):
    """Rows 0 .. most - 1 are the prompts', the next `seqs` ones the single tokens'."""

    def __init__(self, N, dtype, seqs, most):
        super().__init__(N, dtype, seqs, most + seqs)
        self.most = most
        self.parts_of = []  # of the prompts and of the tokens: what is asked for, starts, served
        for _ in range(2):
            self.parts_of.append(tuple(torch.zeros(n, dtype=torch.int32, device="cuda") for n in (seqs, seqs + 1, seqs)))
        self.q_seq, self.o_seq = (torch.zeros((seqs, HEADS * DIM), dtype=self.x.dtype, device="cuda") for _ in range(2))

    def assign(self, part, first, tokens):
        new, starts, served = self.parts_of[part]
        a = self.N.KvAssignDesc(seqs=self.seqs, page_size=PAGE, n_pages=PAGES, max_pages=ROW, max_tokens=tokens)
        state = (self.lengths, self.next, self.held, self.count)
        self.N.check(self.L.spinn_hip_kv_assign(C.byref(a), ptr(new), *map(ptr, state), ptr(self.free), ptr(self.table), *map(ptr, state), ptr(starts),
                                                ptr(served), ptr(self.seq[first:]), ptr(self.slot[first:]), ptr(self.position[first:]), stream()), "assign")

    def rows_to(self, dst, src, parents):
        """Row i of dst = row parents[i] of src, where there is one."""
        size = HEADS * DIM * src.element_size()
        s = self.N.BeamState(src=src.data_ptr(), dst=dst.data_ptr(), row_bytes=size, src_stride=src.stride(0) * src.element_size(),
                             dst_stride=dst.stride(0) * dst.element_size())
        self.N.check(self.L.spinn_hip_beam_reorder(C.byref(s), 1, 1, src.shape[0], dst.shape[0], ptr(parents), stream()), "rows")

    def step(self):
        N, L, most, rows = self.N, self.L, self.most, self.max_tokens
        self.assign(0, 0, most)
        self.assign(1, most, self.seqs)
        d = self.linear_desc(rows)
        N.check(L.spinn_hip_quantize_rows(self.dtype, rows, WIDTH, ptr(self.x), WIDTH, ptr(self.xq), WIDTH, ptr(self.xs), stream()), "quantize")
        N.check(L.spinn_hip_linear_i8(C.byref(d), ptr(self.xq), ptr(self.xs), ptr(self.packed), ptr(self.ws), None, None, ptr(self.rows),
                                      *self.space("linear", L.spinn_hip_linear_i8_workspace_size(C.byref(d))), stream()), "linear")
        N.check(L.spinn_hip_rope(C.byref(self.rope), rows, ptr(self.position), ptr(self.turns), ptr(self.rows), ptr(self.rows), stream()), "rope")
        q, k, v = self.rows[:, :HEADS * DIM], self.rows[:, HEADS * DIM:(HEADS + KV) * DIM], self.rows[:, (HEADS + KV) * DIM:]
        N.check(L.spinn_hip_kv_append(C.byref(self.kv), rows, ptr(self.seq), ptr(self.slot), ptr(self.position), ptr(k), self.n, ptr(v), self.n,
                                      ptr(self.table), ptr(self.k), ptr(self.v), None, None, 0, stream()), "append")
        p = N.PromptAttentionDesc(dtype=self.dtype, seqs=self.seqs, heads=HEADS, kv_heads=KV, head_dim=DIM, causal=1, q_rows=most, kv_rows=most,
                                  scale=DIM ** -0.5, q_stride=self.n, k_stride=self.n, v_stride=self.n, o_stride=HEADS * DIM)
        N.check(L.spinn_hip_prompt_attention(C.byref(p), ptr(q), ptr(k), ptr(v), ptr(self.parts_of[0][1]), None, ptr(self.o), None,
                                             *self.space("prompt", L.spinn_hip_prompt_attention_workspace_size(C.byref(p))), stream()), "prompt")
        self.rows_to(self.q_seq, q[most:], self.parts_of[1][1])
        a = N.KvAttentionDesc(kv=self.kv, heads=HEADS, max_len=SLOTS, scale=DIM ** -0.5, q_stride=HEADS * DIM, o_stride=HEADS * DIM)
        N.check(L.spinn_hip_kv_attention(C.byref(a), ptr(self.q_seq), ptr(self.k), ptr(self.v), ptr(self.table), ptr(self.lengths), None, None, None,
                                         ptr(self.o_seq), None, *self.space("attend", L.spinn_hip_kv_attention_workspace_size(C.byref(a))), stream()), "attend")
        self.rows_to(self.o[most:], self.o_seq, self.seq[most:])


STEPS = [  # what each of six requests does: brings a prompt, a token ("t"), nothing, or ends
    [40, 0, 17, 0, 1, 0],
    ["t", 0, "t", 90, "t", 0],
    [0, 30, "t", "t", -1, 0],        # an idle one, an ended one, a prompt among tokens
    ["t", "t", -1, 0, 0, 60],
    ["t", -1, 8, "t", 21, "t"],
    [0, 0, "t", "t", 0, 0],
    [-1, 5, -1, -1, "t", -1],
    [0, "t", 77, 0, "t", 0]]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("captured", [False, True], ids=["eager", "captured"])
def test_mixed_steps(hip, dtype, captured):
    """Every row's result against the exact one on the keys and values that its sequence has had so far; rows of no token stay as they were."""
    srv = Mixed(hip, dtype, 6, 100)
    g = gen(4)
    history = {}
    graph = None
    if captured:
        srv.step()  # nothing asked for: workspaces are there
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            srv.step()
    for number, step in enumerate(STEPS):
        prompts = [0 if n == "t" else n for n in step]
        tokens = [int(n == "t") for n in step]
        for (new, _, _), asked in zip(srv.parts_of, (prompts, tokens)):
            new.copy_(torch.tensor(asked, dtype=torch.int32))
        srv.x.copy_(randn(g, srv.max_tokens, WIDTH, dtype=dtype))
        srv.o.fill_(7.0)
        graph.replay() if captured else srv.step()
        torch.cuda.synchronize()
        assert all(served.tolist() == [1] * 6 for _, _, served in srv.parts_of)
        rows, at = {}, 0
        for s, n in enumerate(prompts):
            if n < 0:
                history.pop(s, None)
            if n > 0:
                rows[s] = range(at, at + n)
                at += n
        for i, s in enumerate(s for s in range(6) if tokens[s]):
            rows[s] = [srv.most + i]
        used = torch.zeros(srv.max_tokens, dtype=torch.bool)
        for s, mine in rows.items():
            for r in mine:
                used[r] = True
                row = srv.rows[r].double().cpu()
                past = history.setdefault(s, [])
                past.append((row[HEADS * DIM:(HEADS + KV) * DIM].view(KV, DIM), row[(HEADS + KV) * DIM:].view(KV, DIM)))
                ks, vs = torch.stack([a for a, _ in past], 1), torch.stack([b for _, b in past], 1)
                q = row[:HEADS * DIM].view(KV, HEADS // KV, DIM)
                p = torch.softmax((q @ ks.transpose(1, 2).contiguous()) * DIM ** -0.5, -1)
                close(srv.o[r].cpu(), (p @ vs).reshape(-1), f"step {number}, sequence {s}, token {len(past)}")
                assert int(srv.position[r]) == len(past) - 1
        assert (srv.o.cpu()[~used] == 7).all()
        assert srv.lengths.tolist() == [len(history.get(s, [])) for s in range(6)]

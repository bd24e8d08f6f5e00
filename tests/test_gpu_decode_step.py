"""The decoding step's operators together, as a program that generates runs them: fused projection, append,
attention, output projection with its residual, a wide layer, logits, beam search with its states reordered;
greedy generation with eviction; the step captured into a graph and on other streams.

Everything is compared with the same program in 64 bits. Two layers of fp32 products of at most 128 terms lie between a
step's state and its logits: with every product within 2 (128 + 4) 2^-24 = 1.6e-5 of its terms' magnitudes, and those
under 3, ten of them stay under 5e-4 per step; keys that decide are further apart in these inputs or
equal by construction."""
import ctypes as C

import pytest
import torch

from tests.decodeops import F32, evict_ref, gen, linear_pack, ptr, stream, workspace

pytestmark = pytest.mark.gpu

D, HEADS, KV, DIM, WIDE, VOCAB = 64, 4, 2, 16, 128, 97
ROW = (HEADS + 2 * KV) * DIM


class Weights:
    def __init__(self, seed):
        g = gen(seed)
        r = lambda *s: torch.randn(s, generator=g)
        self.embed = r(VOCAB, D) * 0.7
        self.qkv, self.qkv_b = r(ROW, D) * D ** -0.5, r(ROW) * 0.1
        self.out = r(D, HEADS * DIM) * (HEADS * DIM) ** -0.5
        self.up, self.up_b = r(D, WIDE) * D ** -0.5, r(WIDE) * 0.1  # [K, N], as a MatMul node holds it
        self.down = r(D, WIDE) * WIDE ** -0.5
        self.head = r(VOCAB, D) * 0.4


class Step:
    """One step on the device: buffers, descriptors and packed weights as a program keeps them."""

    def __init__(self, N, w, seqs, page, slots, accumulate=False, beams=1, batch=None, k=None):
        self.N, self.L = N, N.lib()
        self.seqs, self.page = seqs, page
        self.pages = -(-slots // page)
        self.slots = self.pages * page
        z = lambda *s, t=torch.float32: torch.zeros(s, device="cuda", dtype=t)
        self.keep = []

        def lin(m, n, k, wt, act=0, trans_w=1, ldx=0, bias=None):
            d = N.LinearDesc(m=m, n=n, k=k, dtype=F32, trans_w=trans_w, act=act, ldx=ldx)
            packed = linear_pack(N, d, wt.cuda())
            size = self.L.spinn_hip_linear_workspace_size(C.byref(d))
            return d, packed, None if bias is None else bias.cuda(), workspace(size), size

        self.embed = w.embed.cuda()
        self.l_qkv = lin(seqs, ROW, D, w.qkv, bias=w.qkv_b)
        self.l_out = lin(seqs, D, HEADS * DIM, w.out)
        self.l_up = lin(seqs, WIDE, D, w.up, act=N.LINEAR_GELU_TANH, trans_w=0, bias=w.up_b)
        self.l_down = lin(seqs, D, WIDE, w.down)
        self.l_head = lin(seqs, VOCAB, D, w.head)
        self.h, self.qkv, self.o, self.wide = z(seqs, D), z(seqs, ROW), z(seqs, HEADS * DIM), z(seqs, WIDE)
        self.logits = z(seqs, VOCAB)
        n_pages = seqs * self.pages
        self.k, self.v = z(n_pages, KV, page, DIM), z(n_pages, KV, page, DIM)
        self.table = torch.arange(n_pages, device="cuda", dtype=torch.int32).view(seqs, self.pages).clone()
        self.lengths, self.slot = z(seqs, t=torch.int32), z(seqs, t=torch.int32)
        self.position = z(seqs, t=torch.int32)
        self.acc, self.pos = z(seqs, KV, self.slots), z(seqs, KV, self.slots, t=torch.int32)
        kv = N.KvDesc(dtype=F32, seqs=seqs, kv_heads=KV, head_dim=DIM, page_size=page, n_pages=n_pages,
                      max_pages=self.pages, page_stride=KV * page * DIM, head_stride=page * DIM, slot_stride=DIM)
        self.kv = kv
        self.att = N.KvAttentionDesc(kv=kv, heads=HEADS, max_len=self.slots, scale=DIM ** -0.5, accumulate=int(accumulate),
                                     q_stride=ROW, o_stride=HEADS * DIM, acc_stride=self.slots)
        self.att_ws = workspace(self.L.spinn_hip_kv_attention_workspace_size(C.byref(self.att)))
        if batch:
            self.beam = N.BeamDesc(dtype=F32, batch=batch, beams=beams, vocab=VOCAB, k=k, end_token=1, logits_stride=VOCAB)
            self.beam_ws = workspace(self.L.spinn_hip_beam_select_workspace_size(C.byref(self.beam)))
            self.scores, self.next_scores = z(batch, beams), z(batch, k)
            self.parents, self.tokens = z(batch, k, t=torch.int32), z(batch, k, t=torch.int32)
            self.finished = z(batch, beams, t=torch.uint8)
            self.next_table, self.next_finished = torch.zeros_like(self.table), torch.zeros_like(self.finished)

    def _linear(self, l, x, y, res=None):
        d, packed, bias, ws, size = l
        self.N.check(self.L.spinn_hip_linear(C.byref(d), ptr(x), ptr(packed), ptr(bias), ptr(res), ptr(y), ptr(ws), size,
                                             stream()), "linear")

    def forward(self):
        """h -> logits; appends at `slot` first."""
        L, N = self.L, self.N
        self._linear(self.l_qkv, self.h, self.qkv)
        at = lambda i: C.c_void_p(self.qkv.data_ptr() + 4 * i * DIM)
        N.check(L.spinn_hip_kv_append(C.byref(self.kv), self.seqs, None, ptr(self.slot), ptr(self.position), at(HEADS), ROW,
                                      at(HEADS + KV), ROW, ptr(self.table), ptr(self.k), ptr(self.v), ptr(self.acc),
                                      ptr(self.pos), self.slots, stream()), "append")
        acc = ptr(self.acc) if self.att.accumulate else None
        N.check(L.spinn_hip_kv_attention(C.byref(self.att), ptr(self.qkv), ptr(self.k), ptr(self.v), ptr(self.table),
                                         ptr(self.lengths), None, acc, acc, ptr(self.o), None, ptr(self.att_ws),
                                         0 if self.att_ws is None else self.att_ws.numel(), stream()), "attention")
        self._linear(self.l_out, self.o, self.h, res=self.h)  # in place on the residual stream
        self._linear(self.l_up, self.h, self.wide)
        self._linear(self.l_down, self.wide, self.h, res=self.h)
        self._linear(self.l_head, self.h, self.logits)

    def select(self):
        N, L = self.N, self.L
        N.check(L.spinn_hip_beam_select(C.byref(self.beam), ptr(self.logits), ptr(self.scores), ptr(self.finished),
                                        ptr(self.next_scores), ptr(self.parents), ptr(self.tokens), ptr(self.beam_ws),
                                        self.beam_ws.numel(), stream()), "select")
        row = 4 * self.pages
        states = (N.BeamState * 2)(N.BeamState(ptr(self.table), ptr(self.next_table), row, row, row),
                                   N.BeamState(ptr(self.finished), ptr(self.next_finished), 1, 1, 1))
        N.check(L.spinn_hip_beam_reorder(states, 2, self.beam.batch, self.beam.beams, self.beam.k, ptr(self.parents), stream()),
                "reorder")


def ref_forward(w, h, cache, new):
    """The same in 64 bits on lists of rows: cache[s] = [(k [KV, DIM], v [KV, DIM])]; appends `new`'s rows. Returns
    (logits, weights that each slot received [s][KV, len])."""
    f = lambda t: t.double()
    qkv = h @ f(w.qkv).t() + f(w.qkv_b)
    o, weights = torch.zeros(h.shape[0], HEADS * DIM, dtype=torch.float64), []
    for s in range(h.shape[0]):
        q = qkv[s, :HEADS * DIM].view(HEADS, DIM)
        new(cache[s], (qkv[s, HEADS * DIM:(HEADS + KV) * DIM].view(KV, DIM), qkv[s, (HEADS + KV) * DIM:].view(KV, DIM)))
        k, v = torch.stack([c[0] for c in cache[s]]), torch.stack([c[1] for c in cache[s]])
        got = torch.zeros(KV, len(cache[s]), dtype=torch.float64)
        for i in range(HEADS):
            g = i // (HEADS // KV)
            p = torch.softmax(k[:, g] @ q[i] * DIM ** -0.5, 0)
            o[s, i * DIM:(i + 1) * DIM] = p @ v[:, g]
            got[g] += p
        weights.append(got)
    h = h + o @ f(w.out).t()
    h = h + torch.nn.functional.gelu(h @ f(w.up) + f(w.up_b), approximate="tanh") @ f(w.down).t()
    return h @ f(w.head).t(), weights


def test_beam_search_over_shared_pages(hip, torch_gpu):
    """Beams share the pages of their common past: pages of one slot, so that a reordered table is all that a
    beam's cache needs; ended beams stay as they are."""
    N, w = hip, Weights(1)
    batch, beams, steps = 2, 3, 9
    seqs = batch * beams
    st = Step(N, w, seqs, 1, steps, batch=batch, beams=beams, k=beams)
    # page p of step t and row s is its own
    fresh = torch.arange(seqs * steps, dtype=torch.int32).view(seqs, steps)
    st.table.fill_(-1)
    tokens = torch.tensor([[5] * beams, [9] * beams])
    scores = torch.tensor([[0.0] + [-float("inf")] * (beams - 1)] * batch)
    st.scores.copy_(scores)
    cache, ref_scores, ref_tokens = [[] for _ in range(seqs)], scores.double(), tokens.clone()
    ref_done = torch.zeros(batch, beams, dtype=torch.bool)
    for t in range(steps):
        # device
        st.table[:, t] = fresh[:, t].cuda()
        st.h.copy_(st.embed[tokens.flatten().cuda()])
        st.slot.fill_(t)
        st.position.fill_(t)
        st.lengths.fill_(t + 1)
        st.forward()
        st.select()
        tokens = st.tokens.cpu().long()
        st.scores.copy_(st.next_scores)
        st.table.copy_(st.next_table)
        st.finished.copy_(st.next_finished)
        st.finished |= (st.tokens == 1).to(torch.uint8)
        # reference
        logits, _ = ref_forward(w, w.embed.double()[ref_tokens.flatten()], cache, lambda c, r: c.append(r))
        logp = torch.log_softmax(logits, 1).view(batch, beams, VOCAB)
        only = torch.full((VOCAB,), -float("inf"), dtype=torch.float64)
        only[1] = 0.0
        key = ref_scores[:, :, None] + torch.where(ref_done[:, :, None], only, logp)
        val, at = torch.sort(key.view(batch, -1), dim=1, descending=True, stable=True)
        val, par, tok = val[:, :beams], at[:, :beams] // VOCAB, at[:, :beams] % VOCAB
        assert torch.equal(st.parents.cpu().long(), par) and torch.equal(tokens, tok), t
        assert (st.next_scores.cpu().double() - val).abs().max() <= 5e-4 * (t + 1)
        cache = [list(cache[b * beams + int(par[b, j])]) for b in range(batch) for j in range(beams)]
        ref_done = torch.gather(ref_done, 1, par) | (tok == 1)
        ref_scores, ref_tokens = val, tok
        assert torch.equal(st.finished.cpu().bool(), ref_done)


def test_generation_with_eviction(hip, torch_gpu):
    """Greedy generation of ragged sequences; every step's weights accumulate, and a cache over its budget is cut."""
    N, w = hip, Weights(2)
    seqs, budget, recent, sinks, steps = 3, 12, 4, 1, 40
    st = Step(N, w, seqs, 8, 24, accumulate=True)
    d = N.KvEvictDesc(kv=st.kv, budget=budget, recent=recent, sinks=sinks, max_len=st.slots, acc_stride=st.slots)
    ws = workspace(st.L.spinn_hip_kv_evict_workspace_size(C.byref(d)))
    cache, lens = [[] for _ in range(seqs)], [0] * seqs
    acc = torch.zeros(seqs, KV, st.slots, dtype=torch.float64)
    pos = torch.zeros(seqs, KV, st.slots, dtype=torch.int32)
    tokens = torch.tensor([3, 20, 50])

    class Heads:  # evict_ref wants the cache's sizes alone
        kv = KV
    Heads.seqs = seqs
    for t in range(steps):
        st.h.copy_(st.embed[tokens.cuda()])
        st.slot.copy_(torch.tensor(lens, dtype=torch.int32))
        st.position.fill_(t)
        st.lengths.copy_(torch.tensor([n + 1 for n in lens], dtype=torch.int32))
        st.forward()
        # the reference's rows of every kv head by themselves: they are evicted by themselves
        ref, weights = ref_forward(w, w.embed.double()[tokens], cache, lambda c, r: c.append((r[0].clone(), r[1].clone())))
        assert (st.logits.cpu().double() - ref).abs().max() <= 5e-4, t
        for s in range(seqs):
            acc[s, :, lens[s]], pos[s, :, lens[s]] = 0, t
            lens[s] += 1
            acc[s, :, :lens[s]] += weights[s]
        got = st.acc.cpu().double()
        for s in range(seqs):
            assert (got[s, :, :lens[s]] - acc[s, :, :lens[s]]).abs().max() <= 5e-4 * (t + 1)
        if t % 5 == 4:  # cut to the budget, those over it
            nxt = torch.full((seqs,), t + 1, dtype=torch.int32).cuda()
            N.check(st.L.spinn_hip_kv_evict(C.byref(d), ptr(st.table), ptr(st.lengths), ptr(nxt), ptr(st.acc), ptr(st.pos), ptr(st.acc),
                                            ptr(st.pos), ptr(st.lengths), ptr(st.k), ptr(st.v), ptr(ws), ws.numel(), stream()), "evict")
            moves, wa, wp, lens = evict_ref(Heads, lens, [t + 1] * seqs, got, pos, budget, recent, sinks, st.slots)
            assert st.lengths.tolist() == lens
            for s, h, frm, to in moves:
                cache[s][to][0][h], cache[s][to][1][h] = cache[s][frm][0][h].clone(), cache[s][frm][1][h].clone()
            for (s, h), a in wa.items():
                acc[s, h, :len(a)], pos[s, h, :len(a)] = torch.tensor(a), torch.tensor(wp[s, h], dtype=torch.int32)
                assert st.pos[s, h, :len(a)].tolist() == wp[s, h]
            cache = [c[:n] for c, n in zip(cache, lens)]
        tokens = ref.argmax(1)


def _fill(st, g, t):
    st.h.copy_(torch.randn(st.seqs, D, generator=g))
    st.slot.fill_(t)
    st.position.fill_(t)
    st.lengths.copy_(torch.randint(0, t + 2, (st.seqs,), generator=g))
    st.scores.copy_(-torch.rand(st.scores.shape, generator=g))


def _state(st):
    return [t.clone() for t in (st.logits, st.o, st.k, st.v, st.acc, st.pos, st.next_scores, st.parents, st.tokens, st.next_table)]


@pytest.mark.parametrize("seqs", [4, 80])
def test_step_in_a_graph(hip, torch_gpu, seqs):
    """The captured step, replayed over inputs that change in place, with eager steps and synchronizations between the
    replays, gives every eager step's bits; two graphs over the same workspaces, one after the other."""
    torch = torch_gpu
    N, w = hip, Weights(3)
    make = lambda: Step(N, w, seqs, 16, 300, accumulate=True, batch=seqs // 4, beams=4, k=4)
    a, b = make(), make()  # a runs from graphs, b eagerly
    _fill(a, gen(0), 0)
    a.forward()
    a.select()
    torch.cuda.synchronize()
    a.k.zero_(), a.v.zero_(), a.acc.zero_(), a.pos.zero_()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for gr in graphs:
        with torch.cuda.graph(gr):
            a.forward()
            a.select()
    a.k.zero_(), a.v.zero_(), a.acc.zero_(), a.pos.zero_()
    for t in range(6):
        _fill(a, gen(10 + t), 40 * t)
        _fill(b, gen(10 + t), 40 * t)
        graphs[t % 2].replay()
        b.forward()
        b.select()
        torch.cuda.synchronize()
        for x, y in zip(_state(a), _state(b)):
            assert torch.equal(x, y), t


def test_eviction_in_a_graph(hip, torch_gpu):
    """Append, attention and eviction captured together, the lengths that eviction leaves on the device read by the next
    replay's calls: every replay gives the eager calls' bits, with host work and synchronizations between."""
    torch = torch_gpu
    N, w = hip, Weights(6)
    seqs, budget = 6, 200
    make = lambda: Step(N, w, seqs, 16, 300, accumulate=True)
    a, b = make(), make()  # a from a graph, b eagerly

    def step(st):
        d = N.KvEvictDesc(kv=st.kv, budget=budget, recent=20, sinks=2, max_len=st.slots, acc_stride=st.slots)
        if not hasattr(st, "evict_ws"):
            st.evict_ws = workspace(st.L.spinn_hip_kv_evict_workspace_size(C.byref(d)))
        st.slot.copy_(st.lengths)
        st.lengths += 1
        st.position += 1
        st.forward()
        N.check(st.L.spinn_hip_kv_evict(C.byref(d), ptr(st.table), ptr(st.lengths), ptr(st.position), ptr(st.acc), ptr(st.pos),
                                        ptr(st.acc), ptr(st.pos), ptr(st.lengths), ptr(st.k), ptr(st.v), ptr(st.evict_ws),
                                        st.evict_ws.numel(), stream()), "evict")

    step(a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a)
    start = torch.tensor([196, 199, 200, 250, 0, 100], dtype=torch.int32)
    for st in (a, b):
        g = gen(40)
        st.k.copy_(torch.randn(st.k.shape, generator=g))
        st.v.copy_(torch.randn(st.v.shape, generator=g))
        st.acc.copy_(torch.rand(st.acc.shape, generator=g))
        st.pos.copy_(torch.arange(st.slots, dtype=torch.int32).expand(st.pos.shape))
        st.lengths.copy_(start)
        st.position.copy_(start)
    want = start.clone()
    for t in range(8):
        for st in (a, b):
            st.h.copy_(torch.randn(seqs, D, generator=gen(50 + t)))
        graph.replay()
        step(b)
        torch.cuda.synchronize()
        want = torch.clamp(want + 1, max=budget)
        assert torch.equal(a.lengths.cpu(), want), t
        for x, y in zip((a.logits, a.o, a.k, a.v, a.acc, a.pos, a.lengths), (b.logits, b.o, b.k, b.v, b.acc, b.pos, b.lengths)):
            assert torch.equal(x, y), t


def test_steps_on_two_streams(hip, torch_gpu):
    """Two programs at once on streams of their own, with buffers of their own."""
    torch = torch_gpu
    N, w = hip, Weights(4)
    make = lambda: Step(N, w, 12, 16, 300, accumulate=True, batch=3, beams=4, k=4)
    both, alone = [make(), make()], [make(), make()]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for t in range(4):
        for i in range(2):
            _fill(both[i], gen(20 + 2 * t + i), 50 * t)
            _fill(alone[i], gen(20 + 2 * t + i), 50 * t)
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                both[i].forward()
                both[i].select()
        torch.cuda.synchronize()
        for i in range(2):
            alone[i].forward()
            alone[i].select()
            torch.cuda.synchronize()
            for x, y in zip(_state(both[i]), _state(alone[i])):
                assert torch.equal(x, y), (t, i)


def test_calls_repeat_their_bits(hip, torch_gpu):
    """The same call twice, with other work between: no result depends on what ran before or on the order of atomics."""
    torch = torch_gpu
    N, w = hip, Weights(5)
    st = Step(N, w, 80, 16, 600, accumulate=True, batch=20, beams=4, k=8)
    st.k.copy_(torch.randn(st.k.shape, generator=gen(1)))
    st.v.copy_(torch.randn(st.v.shape, generator=gen(2)))
    st.next_table = torch.zeros(20 * 8, st.pages, device="cuda", dtype=torch.int32)
    st.next_finished = torch.zeros(20, 8, device="cuda", dtype=torch.uint8)
    first = None
    for i in range(3):
        _fill(st, gen(30), 500)
        st.acc.fill_(0.25)
        st.forward()
        st.select()
        torch.cuda.synchronize()
        now = _state(st)
        if first is None:
            first = now
        for x, y in zip(first, now):
            assert torch.equal(x, y), i
        for ws in (st.att_ws, st.beam_ws):
            ws.fill_(i * 77)

"""spinn_hip_kv_assign on the GPU against the definition, request by request. All results are whole numbers."""
import ctypes as C
import random

import pytest
import torch

from tests.decodeops import ptr, stream
from tests.promptops import assign_ref

pytestmark = pytest.mark.gpu


class State:
    """A server's lists on the host and their copies on the device."""

    def __init__(self, rng, seqs, page, row, free, spare=5, lengths=None):
        self.page, self.row, self.seqs = page, row, seqs
        self.lengths = [rng.randint(0, page * row) for _ in range(seqs)] if lengths is None else lengths
        self.next = [n + rng.choice([0, 0, 7]) for n in self.lengths]
        self.held = [-(-n // page) for n in self.lengths]
        names = list(range(sum(self.held) + free + spare))
        rng.shuffle(names)
        self.table = [[-9] * row for _ in range(seqs)]
        for s in range(seqs):
            for j in range(self.held[s]):
                self.table[s][j] = names.pop()
        self.free = [names.pop() for _ in range(free)] + [-5] * (sum(self.held) + spare)
        self.count = free

    def device(self):
        t = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        return dict(lengths=t(self.lengths), next=t(self.next), held=t(self.held), count=t([self.count]), free=t(self.free), table=t(self.table))

    def step(self, new, max_tokens):
        out = assign_ref(new, self.lengths, self.next, self.held, self.free, self.count, self.table, self.page, max_tokens)
        self.lengths, self.next, self.held, self.count = out["lengths"], out["next"], out["held"], out["count"][0]
        return out


def call(N, st, dev, new, max_tokens, in_place=True, positions=True, next_pos=True):
    d = N.KvAssignDesc(seqs=st.seqs, page_size=st.page, n_pages=len(st.free), max_pages=st.row, max_tokens=max_tokens)
    new = torch.tensor(new, dtype=torch.int32, device="cuda")
    full = lambda n: torch.full((n,), 77, dtype=torch.int32, device="cuda")  # noqa: E731
    out = {n: dev[n] if in_place else torch.full_like(dev[n], 77) for n in ("lengths", "next", "held", "count")}
    for n, k in (("starts", st.seqs + 1), ("served", st.seqs), ("seq", max_tokens + 1), ("slot", max_tokens + 1), ("position", max_tokens + 1)):
        out[n] = full(k)
    p = lambda t, given=True: ptr(t) if given else None  # noqa: E731
    N.check(N.lib().spinn_hip_kv_assign(
        C.byref(d), ptr(new), ptr(dev["lengths"]), p(dev["next"], next_pos), ptr(dev["held"]), ptr(dev["count"]), ptr(dev["free"]),
        ptr(dev["table"]), ptr(out["lengths"]), p(out["next"], next_pos), ptr(out["held"]), ptr(out["count"]), ptr(out["starts"]),
        ptr(out["served"]), ptr(out["seq"]), ptr(out["slot"]), p(out["position"], positions), stream()), "assign")
    return out


def compare(st, dev, out, want, max_tokens, skip=()):
    for n in ("lengths", "next", "held", "count", "starts", "served", "seq", "slot", "position"):
        if n in skip:
            continue
        got = out[n].cpu().tolist()
        if n in ("seq", "slot", "position"):
            assert got[max_tokens] == 77, f"{n}: written behind its end"
            got = got[:max_tokens]
        assert got == want[n], n
    assert dev["table"].cpu().tolist() == st.table
    assert dev["free"].cpu().tolist() == st.free


@pytest.mark.parametrize("in_place", [True, False], ids=["in_place", "apart"])
@pytest.mark.parametrize("seqs,page,row,free,most,max_tokens", [
    (1, 16, 4, 8, 1, 1), (1, 1, 1, 1, 1, 0), (7, 16, 8, 20, 60, 400), (64, 16, 32, 64, 1, 64), (65, 20, 16, 300, 300, 5000),
    (300, 16, 64, 900, 40, 4097), (1024, 8, 8, 500, 5, 4000), (1025, 8, 8, 2000, 9, 9000), (3000, 1, 5, 3000, 3, 6000),
    (2500, 64, 4, 900, 250, 200000)])
def test_steps(hip, seqs, page, row, free, most, max_tokens, in_place):
    """Steps of a server in a row: prompts, single tokens, ended requests, such that do not fit, pages and tokens that run out."""
    rng = random.Random(seqs * 31 + page)
    st = State(rng, seqs, page, row, free)
    dev = st.device()
    for step in range(4):
        new = [rng.choice([0, 1, 1, 1, -1, rng.randint(0, most), -2 if step == 1 else 1, page * row + 1 if step == 2 else 1]) for _ in range(seqs)]
        if step == 3:
            new = [-1] * seqs
        want = st.step(new, max_tokens)
        out = call(hip, st, dev, new, max_tokens, in_place)
        for n in ("lengths", "next", "held", "count"):
            dev[n] = out[n]
        compare(st, dev, out, want, max_tokens)


def test_long_prompts(hip):
    """Prompts of many pages, more than one workgroup's threads."""
    rng = random.Random(5)
    st = State(rng, 3, 16, 8192, 20000, lengths=[0, 100, 0])
    dev = st.device()
    new = [131072, 30001, 100000]
    want = st.step(new, 270000)
    compare(st, dev, call(hip, st, dev, new, 270000), want, 270000)


def test_without_positions(hip):
    """next_pos left out: positions are slots. position left out: not written."""
    rng = random.Random(6)
    for positions in (True, False):
        st = State(rng, 20, 16, 8, 50)
        st.next = list(st.lengths)
        dev = st.device()
        new = [rng.choice([-1, 0, 1, 20]) for _ in range(20)]
        want = st.step(new, 300)
        out = call(hip, st, dev, new, 300, positions=positions, next_pos=False)
        compare(st, dev, out, want, 300, skip=("next",) if positions else ("next", "position"))
        if not positions:
            assert (out["position"] == 77).all()


def test_numbers_out_of_range(hip):
    """Negative lengths count as 0, more pages than a row or free ones than there are as all of them; sums past 32 bits stop."""
    rng = random.Random(7)
    st = State(rng, 6, 16, 4, 10, lengths=[0] * 6)
    st.lengths, st.next, st.held = [-5, 3, 0, 70, 0, 0], [-1, 3, 0, 70, 0, 0], [-3, 1, 0, 9, 0, 0]
    dev = st.device()
    new = [5, 2 ** 31 - 1, 2 ** 31 - 1, 0, 2 ** 31 - 1, -(2 ** 31)]
    want = st.step(new, 40)
    compare(st, dev, call(hip, st, dev, new, 40), want, 40)
    st.count = 10 ** 6
    dev["count"].fill_(10 ** 6)
    new = [1, 1, 0, 0, 3, 1]
    want = st.step(new, 40)
    compare(st, dev, call(hip, st, dev, new, 40), want, 40)


def test_captured_and_replayed(hip):
    """A captured step whose results are its next inputs, replayed with other requests in the same memory."""
    rng = random.Random(8)
    st = State(rng, 40, 16, 32, 500, lengths=[rng.randint(0, 200) for _ in range(40)])
    dev = st.device()
    d = hip.KvAssignDesc(seqs=40, page_size=16, n_pages=len(st.free), max_pages=32, max_tokens=5000)
    new_dev = torch.zeros(40, dtype=torch.int32, device="cuda")
    out = {n: torch.zeros(k, dtype=torch.int32, device="cuda") for n, k in
           (("starts", 41), ("served", 40), ("seq", 5000), ("slot", 5000), ("position", 5000))}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hip.check(hip.lib().spinn_hip_kv_assign(
            C.byref(d), ptr(new_dev), ptr(dev["lengths"]), ptr(dev["next"]), ptr(dev["held"]), ptr(dev["count"]), ptr(dev["free"]), ptr(dev["table"]),
            ptr(dev["lengths"]), ptr(dev["next"]), ptr(dev["held"]), ptr(dev["count"]), *(ptr(out[n]) for n in
                                                                                       ("starts", "served", "seq", "slot", "position")), stream()), "assign")
    for _ in range(6):
        new = [rng.choice([0, 1, 1, 1, -1, rng.randint(1, 150)]) for _ in range(40)]
        new_dev.copy_(torch.tensor(new, dtype=torch.int32))
        want = st.step(new, 5000)
        graph.replay()
        torch.cuda.synchronize()
        for n in ("lengths", "next", "held", "count"):
            assert dev[n].cpu().tolist() == want[n], n
        for n, t in out.items():
            assert t.cpu().tolist() == want[n], n
        assert dev["table"].cpu().tolist() == st.table and dev["free"].cpu().tolist() == st.free

"""What the decoding step's entry points refuse, and what they ask for, without a GPU: every call here
returns before it launches anything."""
import ctypes as C

import pytest

from tests.decodeops import BF16, F16, F32

P = C.c_void_p(4096)  # never dereferenced
ODD = C.c_void_p(4097)
EINVAL, EWORKSPACE = -1, -3
EUNSUPPORTED = -2


def linear_desc(N, **kw):
    a = dict(m=4, n=64, k=64, dtype=BF16, trans_w=1, act=0, x_unaligned=0, reserved=0, ldx=0, ldres=0, ldy=0)
    return N.LinearDesc(**{**a, **kw})


def kv_desc(N, **kw):
    a = dict(dtype=F16, seqs=2, kv_heads=2, head_dim=64, page_size=16, n_pages=8, max_pages=4, reserved=0,
             page_stride=2048, head_stride=1024, slot_stride=64)
    return N.KvDesc(**{**a, **kw})


def test_struct_sizes(native):
    assert [C.sizeof(t) for t in (native.LinearDesc, native.KvDesc, native.KvAttentionDesc, native.KvEvictDesc,
                                  native.BeamDesc, native.BeamState)] == [56, 56, 104, 80, 32, 40]


@pytest.mark.parametrize("bad", [dict(m=-1), dict(n=0), dict(k=0), dict(dtype=2), dict(dtype=11), dict(trans_w=2), dict(act=2),
                                 dict(act=4), dict(act=8), dict(x_unaligned=2), dict(reserved=1), dict(ldx=63), dict(ldres=63),
                                 dict(ldy=-1), dict(ldx=1 << 40)], ids=str)
def test_linear_descriptors(native, bad):
    L = native.lib()
    d = linear_desc(native, **bad)
    assert L.spinn_hip_linear(C.byref(d), P, P, None, None, P, P, 1 << 30, None) == EINVAL
    assert L.spinn_hip_linear_pack_weights(C.byref(d), P, P, None) == EINVAL
    assert L.spinn_hip_linear_packed_size(C.byref(d)) == 0
    assert L.spinn_hip_linear_workspace_size(C.byref(d)) == 0


def test_linear_arguments(native):
    L = native.lib()
    d = linear_desc(native)
    call = lambda *a, d=d: L.spinn_hip_linear(C.byref(d), *a, None)
    assert L.spinn_hip_linear(None, P, P, None, None, P, None, 0, None) == EINVAL
    Q = C.c_void_p(8192)
    for a in ((None, P, None, None, Q), (P, None, None, None, Q), (P, P, None, None, None), (ODD, P, None, None, Q),
              (C.c_void_p(4098), P, None, None, Q), (P, C.c_void_p(4104), None, None, Q), (P, P, ODD, None, Q),
              (P, P, None, ODD, Q), (P, P, None, None, ODD)):
        assert call(*a, None, 0) == EINVAL
    assert call(P, P, None, None, P, None, 0) == EINVAL  # over its own input
    # over its own residual, with another stride
    assert call(P, P, None, Q, Q, None, 0, d=linear_desc(native, ldy=72)) == EINVAL
    assert call(None, None, None, None, None, None, 0, d=linear_desc(native, m=0)) == 0
    # many rows that are no whole 16-byte runs ask for workspace, few do not
    for kw in (dict(k=60), dict(ldx=65), dict(x_unaligned=1)):
        assert L.spinn_hip_linear_workspace_size(C.byref(linear_desc(native, **kw))) == 0
        d2 = linear_desc(native, m=4000, n=4096, **kw)
        size = L.spinn_hip_linear_workspace_size(C.byref(d2))
        assert size > 0
        assert call(P, P, None, None, Q, None, 0, d=d2) == EWORKSPACE
        assert call(P, P, None, None, Q, P, size - 1, d=d2) == EWORKSPACE
        assert call(P, P, None, None, Q, C.c_void_p(4104), size, d=d2) == EWORKSPACE
    # packed weights hold every weight, whatever m and the layout
    for kw in (dict(), dict(n=65), dict(k=1), dict(dtype=F32), dict(m=4000), dict(trans_w=0)):
        d2 = linear_desc(native, **kw)
        assert L.spinn_hip_linear_packed_size(C.byref(d2)) >= d2.n * d2.k * (4 if d2.dtype == F32 else 2)
    assert L.spinn_hip_linear_packed_size(C.byref(linear_desc(native, m=1))) == L.spinn_hip_linear_packed_size(C.byref(linear_desc(native, m=500, trans_w=0)))


KV_BAD = [dict(dtype=7), dict(seqs=-1), dict(kv_heads=0), dict(head_dim=0), dict(head_dim=257), dict(page_size=0), dict(n_pages=0),
          dict(max_pages=0), dict(reserved=1), dict(max_pages=1 << 30, page_size=16), dict(page_stride=63), dict(head_stride=0),
          dict(slot_stride=63), dict(page_stride=1 << 60), dict(slot_stride=-64)]


@pytest.mark.parametrize("bad", KV_BAD, ids=str)
def test_cache_descriptors(native, bad):
    L, N = native.lib(), native
    kv = kv_desc(N, **bad)
    assert L.spinn_hip_kv_append(C.byref(kv), 1, None, P, None, P, 128, P, 128, P, P, P, None, None, 0, None) == EINVAL
    a = N.KvAttentionDesc(kv=kv, heads=4, max_len=16, scale=1, q_stride=1 << 12, o_stride=1 << 12)
    assert L.spinn_hip_kv_attention(C.byref(a), P, P, P, P, P, None, None, None, P, None, P, 1 << 30, None) == EINVAL
    assert L.spinn_hip_kv_attention_workspace_size(C.byref(a)) == 0
    e = N.KvEvictDesc(kv=kv, budget=4, recent=1, sinks=1, max_len=16, acc_stride=64)
    assert L.spinn_hip_kv_evict(C.byref(e), P, P, P, P, P, P, P, P, P, P, P, 1 << 30, None) == EINVAL
    assert L.spinn_hip_kv_evict_workspace_size(C.byref(e)) == 0


def test_append_arguments(native):
    L = native.lib()
    kv = kv_desc(native)

    def call(tokens=2, seq=None, slot=P, k=P, ks=128, v=P, vs=128, table=P, kp=P, vp=P, acc=None, pos=None, stride=0, d=kv):
        return L.spinn_hip_kv_append(C.byref(d), tokens, seq, slot, None, k, ks, v, vs, table, kp, vp, acc, pos, stride, None)

    for kw in (dict(tokens=-1), dict(tokens=3), dict(slot=None), dict(k=None), dict(v=None), dict(table=None), dict(kp=None),
               dict(vp=None), dict(ks=127), dict(vs=0), dict(k=ODD), dict(vp=ODD), dict(acc=P), dict(pos=P, stride=-1)):
        assert call(**kw) == EINVAL, kw
    assert L.spinn_hip_kv_append(None, 0, None, P, None, P, 128, P, 128, P, P, P, None, None, 0, None) == EINVAL
    assert call(tokens=0) == 0
    assert call(tokens=5, seq=P, d=kv_desc(native, seqs=0)) == 0


def test_append_rows_past_31_bits(native):
    """A token's row of all heads is counted in 31 bits: longer ones are refused, not cut short."""
    L = native.lib()
    for kv_heads, head_dim in ((1 << 24, 256), (1 << 23, 256), ((1 << 22) + 1, 256)):
        row = kv_heads * head_dim
        kv = kv_desc(native, kv_heads=kv_heads, head_dim=head_dim, page_size=1, page_stride=row, head_stride=head_dim, slot_stride=head_dim)
        assert L.spinn_hip_kv_append(C.byref(kv), 1, None, P, None, P, row, P, row, P, P, P, None, None, 0, None) == EINVAL


def test_attention_arguments(native):
    L, N = native.lib(), native

    def desc(kv=None, **kw):
        a = dict(heads=4, max_len=64, scale=1.0, accumulate=0, q_stride=256, o_stride=256, mask_stride=64, acc_stride=64)
        return N.KvAttentionDesc(kv=kv or kv_desc(N), **{**a, **kw})

    def call(d=None, q=P, k=P, v=P, table=P, lengths=P, mask=None, acc=None, out=None, o=P, ws=P, size=1 << 30):
        return L.spinn_hip_kv_attention(C.byref(d or desc()), q, k, v, table, lengths, mask, acc, out, o, None, ws, size, None)

    for kw in (dict(heads=0), dict(heads=3), dict(max_len=-1), dict(max_len=65), dict(accumulate=2), dict(q_stride=255),
               dict(o_stride=0), dict(accumulate=1, acc_stride=63), dict(mask_stride=-1)):
        assert call(desc(**kw)) == EINVAL, kw
        assert L.spinn_hip_kv_attention_workspace_size(C.byref(desc(**kw))) == 0
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(table=None), dict(lengths=None), dict(o=None), dict(q=ODD), dict(o=ODD),
               dict(d=desc(mask_stride=63), mask=P), dict(d=desc(accumulate=1)), dict(d=desc(accumulate=1), acc=P)):
        assert call(**kw) == EINVAL, kw
    d = desc(accumulate=1)
    size = L.spinn_hip_kv_attention_workspace_size(C.byref(d))
    assert size >= 2 * 4 * 64 * 4
    assert call(d, acc=P, out=P, ws=None, size=0) == EWORKSPACE
    assert call(d, acc=P, out=P, size=size - 1) == EWORKSPACE
    assert call(d, acc=P, out=P, ws=C.c_void_p(4100), size=size) == EWORKSPACE
    assert call(desc(kv=kv_desc(N, seqs=0))) == 0


def test_evict_arguments(native):
    L, N = native.lib(), native

    def desc(kv=None, **kw):
        a = dict(budget=32, recent=4, sinks=1, max_len=64, acc_stride=64)
        return N.KvEvictDesc(kv=kv or kv_desc(N), **{**a, **kw})

    def call(d=None, args=(P,) * 10, ws=P, size=1 << 30):
        return L.spinn_hip_kv_evict(C.byref(d or desc()), *args, ws, size, None)

    for kw in (dict(budget=-1), dict(recent=-1), dict(sinks=-1), dict(max_len=65), dict(max_len=-1), dict(acc_stride=63)):
        assert call(desc(**kw)) == EINVAL, kw
    for i in range(10):
        assert call(args=(P,) * i + (None,) + (P,) * (9 - i)) == EINVAL, i
    assert call(args=(P,) * 8 + (ODD, P)) == EINVAL
    size = L.spinn_hip_kv_evict_workspace_size(C.byref(desc()))
    assert size > 0 and call(size=size - 1) == EWORKSPACE and call(ws=None) == EWORKSPACE
    assert call(desc(kv=kv_desc(N, seqs=0))) == 0


def test_beam_arguments(native):
    L, N = native.lib(), native

    def desc(**kw):
        a = dict(dtype=F32, batch=2, beams=4, vocab=100, k=8, end_token=0, logits_stride=100)
        return N.BeamDesc(**{**a, **kw})

    def call(d=None, logits=P, scores=P, fin=None, os=P, op=P, ot=P, ws=P, size=1 << 30):
        return L.spinn_hip_beam_select(C.byref(d or desc()), logits, scores, fin, os, op, ot, ws, size, None)

    for kw in (dict(dtype=6), dict(batch=-1), dict(beams=0), dict(beams=65), dict(vocab=0), dict(k=0), dict(k=129),
               dict(vocab=1, k=5, logits_stride=1), dict(logits_stride=99)):
        assert call(desc(**kw)) == EINVAL, kw
        assert L.spinn_hip_beam_select_workspace_size(C.byref(desc(**kw))) == 0
    for kw in (dict(logits=None), dict(scores=None), dict(os=None), dict(op=None), dict(ot=None), dict(logits=C.c_void_p(4098)),
               dict(d=desc(end_token=100), fin=P), dict(d=desc(end_token=-1), fin=P)):
        assert call(**kw) == EINVAL, kw
    size = L.spinn_hip_beam_select_workspace_size(C.byref(desc()))
    assert size > 0 and call(size=size - 1) == EWORKSPACE and call(ws=None) == EWORKSPACE
    assert call(desc(batch=0)) == 0


def test_reorder_arguments(native):
    L, N = native.lib(), native

    def call(states, n=None, batch=2, beams=4, k=4, parents=P):
        arr = (N.BeamState * max(1, len(states)))(*states)
        return L.spinn_hip_beam_reorder(arr, len(states) if n is None else n, batch, beams, k, parents, None)

    A, B = C.c_void_p(1 << 20), C.c_void_p(1 << 21)
    ok = N.BeamState(A, B, 64, 64, 64)
    for s in (N.BeamState(None, B, 64, 64, 64), N.BeamState(A, None, 64, 64, 64), N.BeamState(A, B, -1, 64, 64),
              N.BeamState(A, B, 64, 63, 64), N.BeamState(A, B, 64, 64, 63), N.BeamState(A, A, 64, 64, 64),
              N.BeamState(A, C.c_void_p((1 << 20) + 511), 64, 64, 64)):
        assert call([s]) == EINVAL
    # one state's destination over another's source
    assert call([ok, N.BeamState(B, C.c_void_p(1 << 22), 64, 64, 64)]) == EINVAL
    assert call([ok], parents=None) == EINVAL
    assert call([ok], batch=-1) == EINVAL and call([ok], beams=0) == EINVAL and call([ok], k=0) == EINVAL
    assert call([ok] * 17) == EINVAL and call([ok], n=-1) == EINVAL
    # sizes whose ends would not fit 64 bits
    far = N.BeamState(A, B, 64, 1 << 38, 1 << 38)
    assert call([far], batch=1 << 21, beams=4, k=1) == EINVAL and call([far], batch=1 << 21, k=4) == EINVAL
    assert call([N.BeamState(A, B, 64, (1 << 38) + 64, 64)]) == EINVAL
    assert call([], n=0) == 0 and call([ok], batch=0) == 0


def test_launches_past_32_bits_of_threads(native):
    """Grids of more than 2^32 threads, which the runtime would cut short without an error, are refused before anything runs."""
    L, N = native.lib(), native
    Q = C.c_void_p(8192)
    for kw in (dict(m=1, n=1 << 27), dict(m=1 << 24, n=1 << 24, k=1024)):
        d = linear_desc(N, **kw)
        assert L.spinn_hip_linear(C.byref(d), P, P, None, None, Q, P, 1 << 62, None) == EUNSUPPORTED, kw
    b = N.BeamDesc(dtype=F32, batch=1 << 19, beams=64, vocab=100, k=8, logits_stride=100)
    assert L.spinn_hip_beam_select(C.byref(b), P, P, None, P, P, P, P, 1 << 62, None) == EUNSUPPORTED
    kv = kv_desc(N, dtype=F32, seqs=1 << 14, kv_heads=8, head_dim=256, page_stride=1 << 16, head_stride=4096, slot_stride=256,
                 max_pages=1 << 14)
    a = N.KvAttentionDesc(kv=kv, heads=8, max_len=1 << 18, scale=1.0, q_stride=2048, o_stride=2048)
    assert L.spinn_hip_kv_attention(C.byref(a), P, P, P, P, P, None, None, None, P, None, P, 1 << 62, None) == EUNSUPPORTED
    e = N.KvEvictDesc(kv=kv_desc(N, seqs=1 << 20, kv_heads=8, page_stride=8192), budget=4, recent=1, sinks=1, max_len=16, acc_stride=64)
    assert L.spinn_hip_kv_evict(C.byref(e), P, P, P, P, P, P, P, P, P, P, P, 1 << 62, None) == EUNSUPPORTED

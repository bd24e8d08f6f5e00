"""What the entry points around a prompt refuse, and what they ask for, without a GPU: every call here returns before
it launches anything."""
import ctypes as C

import pytest

from tests.decodeops import BF16, F16, F32

P, Q = C.c_void_p(4096), C.c_void_p(8192)  # never dereferenced
ODD = C.c_void_p(4097)
EINVAL, EUNSUPPORTED, EWORKSPACE = -1, -2, -3


def test_struct_sizes(native):
    N = native
    assert [C.sizeof(t) for t in (N.KvAssignDesc, N.RopeDesc, N.PromptAttentionDesc, N.LinearI8Desc)] == [24, 80, 72, 48]


# ---- pages ----

def assign_desc(N, **kw):
    return N.KvAssignDesc(**{**dict(seqs=4, page_size=16, n_pages=64, max_pages=8, max_tokens=128, reserved=0), **kw})


@pytest.mark.parametrize("bad", [dict(seqs=-1), dict(seqs=65537), dict(page_size=0), dict(n_pages=0), dict(n_pages=(1 << 29) + 1),
                                 dict(max_pages=0), dict(max_tokens=-1), dict(max_tokens=(1 << 28) + 1), dict(reserved=1),
                                 dict(page_size=1 << 16, max_pages=1 << 16)], ids=str)
def test_assign_descriptors(native, bad):
    assert native.lib().spinn_hip_kv_assign(C.byref(assign_desc(native, **bad)), *(P,) * 16, None) == EINVAL


def test_assign_arguments(native):
    L = native.lib()
    d = assign_desc(native)
    optional = {2, 8, 15}  # next_pos and next_out together, position
    for i in range(16):
        a = [P] * 16
        a[i] = None
        if i == 8 or i not in optional:
            assert L.spinn_hip_kv_assign(C.byref(d), *a, None) == EINVAL, i
    assert L.spinn_hip_kv_assign(None, *(P,) * 16, None) == EINVAL
    assert L.spinn_hip_kv_assign(C.byref(assign_desc(native, seqs=0)), *(None,) * 16, None) == 0


# ---- rotary positions ----

def rope_desc(N, **kw):
    a = dict(dtype=BF16, heads=4, head_dim=64, rot_dim=64, interleaved=0, scaling=0, base=10000.0, factor=1.0, low=1.0, high=4.0,
             trained=2048, magnitude=1.0, x_stride=256, x_head_stride=64, y_stride=256, y_head_stride=64)
    return N.RopeDesc(**{**a, **kw})


NAN, INF = float("nan"), float("inf")
ROPE_TABLE_BAD = [dict(rot_dim=0), dict(rot_dim=63), dict(rot_dim=514, head_dim=600), dict(scaling=3), dict(scaling=-1), dict(base=0.0),
                  dict(base=NAN), dict(base=-2.0), dict(factor=2.0), dict(scaling=1, factor=0.0), dict(scaling=1, factor=INF),
                  dict(scaling=2, trained=0), dict(scaling=2, low=4.0), dict(scaling=2, high=NAN)]
ROPE_BAD = ROPE_TABLE_BAD + [dict(dtype=2), dict(heads=0), dict(rot_dim=66), dict(head_dim=513), dict(interleaved=2), dict(magnitude=NAN),
                             dict(x_stride=63), dict(y_stride=-256), dict(x_head_stride=63), dict(y_head_stride=1 << 33),
                             dict(heads=1 << 25)]


@pytest.mark.parametrize("bad", ROPE_BAD, ids=str)
def test_rope_descriptors(native, bad):
    L = native.lib()
    d = rope_desc(native, **bad)
    assert L.spinn_hip_rope(C.byref(d), 1, P, P, P, Q, None) == EINVAL
    if bad in ROPE_TABLE_BAD:
        assert L.spinn_hip_rope_table_size(C.byref(d)) == 0
        assert L.spinn_hip_rope_table(C.byref(d), P, None) == EINVAL


def test_rope_arguments(native):
    L = native.lib()
    d = rope_desc(native)
    assert L.spinn_hip_rope_table_size(C.byref(d)) == 32 * 8
    for t in (None, C.c_void_p(4104)):
        assert L.spinn_hip_rope_table(C.byref(d), t, None) == EINVAL
    call = lambda *a, d=d: L.spinn_hip_rope(C.byref(d), *a, None)  # noqa: E731
    for a in ((-1, P, P, P, Q), ((1 << 28) + 1, P, P, P, Q), (1, None, P, P, Q), (1, P, None, P, Q), (1, P, C.c_void_p(4104), P, Q),
              (1, P, P, None, Q), (1, P, P, P, None), (1, P, P, ODD, Q), (1, P, P, P, ODD)):
        assert call(*a) == EINVAL, a
    assert call(1, P, P, P, P, d=rope_desc(native, y_stride=512)) == EINVAL  # in place with other strides
    assert call(0, None, None, None, None) == 0


# ---- attention ----

def prompt_desc(N, **kw):
    a = dict(dtype=F16, seqs=2, heads=4, kv_heads=2, head_dim=64, causal=1, q_rows=100, kv_rows=100, scale=0.125, reserved=0,
             q_stride=512, k_stride=512, v_stride=512, o_stride=256)
    return N.PromptAttentionDesc(**{**a, **kw})


@pytest.mark.parametrize("bad", [dict(dtype=7), dict(seqs=-1), dict(seqs=(1 << 24) + 1), dict(heads=0), dict(heads=3), dict(kv_heads=0),
                                 dict(head_dim=0), dict(head_dim=257), dict(causal=2), dict(causal=-1), dict(q_rows=-1), dict(kv_rows=-1),
                                 dict(scale=NAN), dict(scale=INF), dict(reserved=1), dict(q_stride=255), dict(k_stride=127),
                                 dict(v_stride=-1), dict(o_stride=255), dict(q_stride=(1 << 24) + 1), dict(q_rows=1 << 29, kv_rows=1 << 29)], ids=str)
def test_prompt_descriptors(native, bad):
    L = native.lib()
    d = prompt_desc(native, **bad)
    assert L.spinn_hip_prompt_attention(C.byref(d), P, P, P, P, P, Q, None, P, 1 << 40, None) == EINVAL
    assert L.spinn_hip_prompt_attention_workspace_size(C.byref(d)) == 0


def test_prompt_arguments(native):
    L = native.lib()

    def call(d=None, q=P, k=P, v=P, starts=P, kv=None, o=Q, lse=None, ws=P, size=1 << 40):
        return L.spinn_hip_prompt_attention(C.byref(d or prompt_desc(native)), q, k, v, starts, kv, o, lse, ws, size, None)

    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(starts=None), dict(o=None), dict(o=P), dict(q=ODD), dict(k=ODD), dict(v=ODD),
               dict(o=ODD), dict(d=prompt_desc(native, kv_rows=50))):
        assert call(**kw) == EINVAL, kw
    assert L.spinn_hip_prompt_attention(None, P, P, P, P, None, Q, None, P, 0, None) == EINVAL
    nothing = dict(q=None, k=None, v=None, starts=None, o=None, ws=None, size=0)
    assert call(prompt_desc(native, seqs=0), **nothing) == 0
    assert call(prompt_desc(native, q_rows=0, kv_rows=0), **nothing) == 0
    # the workspace that a call asks for is demanded
    for kw in (dict(), dict(q_rows=4000, kv_rows=4000), dict(q_rows=16, kv_rows=100000)):
        d = prompt_desc(native, **kw)
        size = L.spinn_hip_prompt_attention_workspace_size(C.byref(d))
        if size:
            assert call(d, kv=P, size=size - 1) == EWORKSPACE and call(d, kv=P, ws=None) == EWORKSPACE
            assert call(d, kv=P, ws=C.c_void_p(4100)) == EWORKSPACE


# ---- 8-bit linear layers ----

def i8_desc(N, **kw):
    return N.LinearI8Desc(**{**dict(m=4, n=64, k=64, dtype=BF16, trans_w=1, act=0, ldx=0, ldres=0, ldy=0), **kw})


@pytest.mark.parametrize("bad", [dict(m=-1), dict(n=0), dict(k=0), dict(k=131072), dict(dtype=3), dict(trans_w=2), dict(act=2), dict(act=8),
                                 dict(ldx=48), dict(ldx=72), dict(k=65, ldx=64), dict(ldres=63), dict(ldy=-1), dict(ldx=1 << 40)], ids=str)
def test_linear_i8_descriptors(native, bad):
    L = native.lib()
    d = i8_desc(native, **bad)
    assert L.spinn_hip_linear_i8(C.byref(d), P, P, P, P, None, None, Q, P, 1 << 30, None) == EINVAL
    assert L.spinn_hip_linear_i8_pack_weights(C.byref(d), P, P, None) == EINVAL
    assert L.spinn_hip_linear_i8_packed_size(C.byref(d)) == 0
    assert L.spinn_hip_linear_i8_workspace_size(C.byref(d)) == 0


def test_linear_i8_arguments(native):
    L = native.lib()
    d = i8_desc(native)
    call = lambda *a, d=d: L.spinn_hip_linear_i8(C.byref(d), *a, None)  # noqa: E731
    good = (P, P, P, P, None, None, Q)
    for i in (0, 1, 2, 3, 6):
        assert call(*(None if j == i else v for j, v in enumerate(good)), None, 0) == EINVAL, i
    for i, p in ((0, C.c_void_p(4104)), (1, C.c_void_p(4098)), (2, C.c_void_p(4104)), (3, C.c_void_p(4098)), (4, ODD), (5, ODD), (6, ODD),
                 (6, P)):
        assert call(*(p if j == i else v for j, v in enumerate(good)), None, 0) == EINVAL, (i, p)
    assert call(P, P, P, P, None, Q, Q, None, 0, d=i8_desc(native, ldy=72)) == EINVAL  # over its residual, other strides
    assert call(*(None,) * 7, None, 0, d=i8_desc(native, m=0)) == 0
    for kw in (dict(), dict(n=65), dict(k=1), dict(m=4000), dict(trans_w=0)):
        d2 = i8_desc(native, **kw)
        assert L.spinn_hip_linear_i8_packed_size(C.byref(d2)) >= d2.n * d2.k
    d2 = i8_desc(native, m=200, n=1024, k=16384)
    size = L.spinn_hip_linear_i8_workspace_size(C.byref(d2))
    assert size > 0
    assert call(*good, None, 0, d=d2) == EWORKSPACE and call(*good, P, size - 1, d=d2) == EWORKSPACE
    assert call(*good, C.c_void_p(4104), size, d=d2) == EWORKSPACE


def test_quantize_arguments(native):
    L = native.lib()

    def call(dtype=F32, rows=2, k=33, x=P, ldx=33, xq=Q, ldq=48, scale=P):
        return L.spinn_hip_quantize_rows(dtype, rows, k, x, ldx, xq, ldq, scale, None)

    for kw in (dict(dtype=3), dict(rows=-1), dict(k=0), dict(ldx=32), dict(ldq=32), dict(ldq=40), dict(ldx=(1 << 28) + 1), dict(ldq=(1 << 28) + 16), dict(x=None), dict(xq=None), dict(scale=None),
               dict(x=ODD), dict(xq=C.c_void_p(8200))):
        assert call(**kw) == EINVAL, kw
    assert call(rows=0, x=None, xq=None, scale=None) == 0


def test_launches_past_32_bits_of_threads(native):
    L, N = native.lib(), native
    assert L.spinn_hip_quantize_rows(F32, 1 << 30, 5000, P, 5000, Q, 5008, P, None) == EUNSUPPORTED
    d = i8_desc(N, m=1, n=1 << 28)
    assert L.spinn_hip_linear_i8(C.byref(d), P, P, P, P, None, None, Q, P, 1 << 62, None) == EUNSUPPORTED
    d = prompt_desc(N, seqs=1 << 24, heads=64, kv_heads=64, q_rows=1 << 24, kv_rows=1 << 24, head_dim=1)
    assert L.spinn_hip_prompt_attention(C.byref(d), P, P, P, P, None, Q, None, P, 1 << 62, None) == EUNSUPPORTED

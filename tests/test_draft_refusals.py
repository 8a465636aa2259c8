"""What the ops on drafted tokens and the int8 KV cache refuse (host logic, on
a runtime without a device): nothing is launched and no output is left."""
import pytest

PRE = """
import pytest
from esolearn_amd._lib import load
INVALID, OOM, RANGE, UNSUPPORTED = 1, 3, 5, 6
def refuse(code, f, *a, **k):
    launches()
    used = F.fake_used()
    try:
        f(*a, **k)
    except E.ScryHipError as e:
        assert e.code == code, (e.code, str(e))
    else:
        raise AssertionError("not refused")
    assert not launches()
    assert F.fake_used() <= used + (64 << 10)
nq, nkv, hd, rows, ms = 4, 2, 64, 5, 100
z = B.zeros
q, k = z(rows * nq * hd), z(rows * nkv * hd)
qkv, fr, w = z(rows * (nq + 2 * nkv) * hd), z(hd // 2), z(hd)
B.set_bf16_mode(True)
half = B.from_vec_with_bf16(np.zeros(rows * nq * hd, np.float32), np.zeros(rows * nq * hd, np.uint16))
B.set_bf16_mode(False)
kc, vc = z(ms * nkv * hd), z(ms * nkv * hd)
c, c2, other = B.kv8_new(ms, nkv, hd), B.kv8_new(ms, nkv, hd), B.kv8_new(ms, nkv, hd - 4)
par = [-1, 0, 0, 2, -2]
"""

CALLS = {
    "qk_norm_rope": """
f = lambda x=qkv, start=(7,), rows=rows, nq=nq, nkv=nkv, hd=hd, fr=fr, **kw: B.qk_norm_rope(x, start, rows, nq, nkv, hd, fr, **kw)
f(q_weight=w, k_weight=w, parents=par)
refuse(INVALID, f, x=q)
refuse(INVALID, f, x=half)
refuse(INVALID, f, fr=w)
refuse(INVALID, f, q_weight=fr)
refuse(INVALID, f, k_weight=fr)
refuse(INVALID, f, nq=0)
refuse(INVALID, f, nq=3)
refuse(INVALID, f, nkv=0)
refuse(INVALID, f, hd=0)
refuse(UNSUPPORTED, f, hd=66)
refuse(UNSUPPORTED, f, hd=260)
refuse(INVALID, f, rows=0)
refuse(INVALID, f, start=())
refuse(INVALID, f, start=[0] * 17)
refuse(RANGE, f, start=[-1])
refuse(RANGE, f, start=[0x7fffffff])
refuse(RANGE, f, start=[(1 << 30) - rows + 1])
f(start=[(1 << 30) - rows])
refuse(UNSUPPORTED, f, rows=1 << 24)
refuse(UNSUPPORTED, f, start=[0] * 16, rows=1 << 20)
refuse(UNSUPPORTED, f, rows=65, parents=[-1] * 65)
for bad in ([0, 0, 0, 0, 0], [-1, 1, 0, 0, 0], [-3, 0, 0, 0, 0], [-1, 0, -2, 2, 0], [-1, 0, 0, 0, 4]):
    refuse(INVALID, f, parents=bad)
for bad in ([-1] * 4, [[-1] * 5] * 2, [[[-1] * 5]]):
    with pytest.raises(ValueError):
        f(parents=bad)
with pytest.raises(ValueError):
    f(start=[0.5])
with pytest.raises(ValueError):
    f(start=[1 << 40])
""",
    "kv8": """
refuse(INVALID, B.kv8_new, 0, nkv, hd)
refuse(INVALID, B.kv8_new, 0x7fffffff, nkv, hd)
refuse(INVALID, B.kv8_new, (1 << 30) + 1, nkv, hd)
refuse(INVALID, B.kv8_new, 10, 0, hd)
refuse(UNSUPPORTED, B.kv8_new, 10, 1, 30)
refuse(UNSUPPORTED, B.kv8_new, 10, 1, 512)
B.kv8_write([c], k, k, [95], rows)
refuse(RANGE, B.kv8_write, [c], k, k, [96], rows)
refuse(RANGE, B.kv8_write, [c], k, k, [-1], rows)
refuse(INVALID, B.kv8_write, [c], k, k, [0], rows - 1)
refuse(INVALID, B.kv8_write, [c], k, q, [0], rows)
refuse(INVALID, B.kv8_write, [c], half, half, [0], rows)
kk = z(2 * rows * nkv * hd)
B.kv8_write([c, c2], kk, kk, [0, 3], rows)
refuse(INVALID, B.kv8_write, [c, c], kk, kk, [0, 50], rows)
refuse(INVALID, B.kv8_write, [c, other], kk, kk, [0, 3], rows)
B.kv8_read([c, c], [0, 90], 10)
refuse(RANGE, B.kv8_read, [c], [0], ms + 1)
refuse(RANGE, B.kv8_read, [c], [0], 0x7fffffff)
refuse(INVALID, B.kv8_read, [c], [0], 0)
refuse(INVALID, B.kv8_read, [], [], 1)
with pytest.raises(ValueError):
    B.kv8_read([c], [0, 1], 1)
B.kv8_keep([c], [36], [[0, 63]])
launches()
B.kv8_keep([c], [98], [[0, 1, -1, 7]])
B.kv8_keep([c], [99], [[-1]])
assert not launches()
refuse(RANGE, B.kv8_keep, [c], [37], [[0, 63]])
for bad in ([[1, 1]], [[2, 1]], [[64]], [[-2]], [[0, -5]]):
    refuse(INVALID, B.kv8_keep, [c], [0], bad)
refuse(INVALID, B.kv8_keep, [c, c], [0, 9], [[1], [1]])
refuse(INVALID, B.kv8_keep, [c], [0], [[-1] * 65])
with pytest.raises(ValueError):
    B.kv8_keep([c], [0], [1, 2])
gone = B.kv8_new(ms, nkv, hd)
gone.free()
gone.free()
refuse(INVALID, B.kv8_write, [gone], k, k, [0], rows)
refuse(INVALID, B.kv8_keep, [gone], [0], [[1]])
""",
    "attention": """
f = lambda q=q, kc=(kc,), vc=(vc,), lens=(50,), rows=rows, nq=nq, nkv=nkv, hd=hd, **kw: \\
    B.tree_attention(q, kc, vc, lens, rows, nq, nkv, hd, 0.1, **kw)
g = lambda q=q, cs=(c,), lens=(50,), rows=rows, nq=nq, **kw: B.kv8_tree_attention(q, cs, lens, rows, nq, 0.1, **kw)
f(lens=[95], parents=par), g(lens=[95], parents=par)
for h in (f, g):
    refuse(INVALID, h, q=k)
    refuse(INVALID, h, q=half)
    refuse(RANGE, h, lens=[96])
    refuse(RANGE, h, lens=[-1])
    refuse(RANGE, h, lens=[0x7fffffff])
    refuse(INVALID, h, rows=0)
    refuse(INVALID, h, nq=3)
    refuse(INVALID, h, nq=0)
    refuse(INVALID, h, parents=[-1, 0, 0, 5, -2])
    refuse(UNSUPPORTED, h, rows=65, parents=[-1] * 65)
    with pytest.raises(ValueError):
        h(lens=[1, 2])
refuse(INVALID, f, kc=[half])
refuse(INVALID, f, nkv=0)
refuse(UNSUPPORTED, f, hd=34)
refuse(RANGE, f, vc=[z(54 * nkv * hd)])
refuse(INVALID, g, cs=[other])
qq = z(2 * rows * nq * hd)
g(q=qq, cs=[c, c], lens=[3, 4])
refuse(INVALID, g, q=qq, cs=[c, other], lens=[3, 4])
""",
    "verify": """
V = 10
p, qd = z((rows + 1) * V), z(rows * V)
tok, u = np.zeros((1, rows), int), np.zeros((1, rows + 1))
def d(p=p, q=qd, tok=tok, u=u, V=V, **kw):
    return B.verify_draft(p, q, tok, u, V, **kw)
def t(p=p, tok=tok, par=par, u=u, V=V):
    return B.verify_tree(p, tok, par, u, V)
for h in (d, t):
    refuse(INVALID, h, p=qd)
    refuse(INVALID, h, p=half)
    refuse(INVALID, h, V=0)
    for x in (1.0, -0.1, np.nan, np.inf):
        v = u.copy(); v[0, 3] = x
        refuse(INVALID, h, u=v)
    for x in (-1, V, 1 << 40):
        v = tok.copy(); v[0, 3] = x
        refuse(RANGE, h, tok=v)
    with pytest.raises(ValueError):
        h(u=u[:, :-1])
    with pytest.raises(ValueError):
        h(tok=tok[0])
refuse(INVALID, d, q=p)
refuse(INVALID, d, counts=[rows + 1])
refuse(INVALID, d, counts=[-1])
with pytest.raises(ValueError):
    d(counts=[1, 1])
with pytest.raises(ValueError):
    d(tok=tok + 0.5)
refuse(UNSUPPORTED, d, p=z(66 * V), q=z(65 * V), tok=np.zeros((1, 65), int), u=np.zeros((1, 66)))
refuse(UNSUPPORTED, t, p=z(66 * V), tok=np.zeros((1, 65), int), par=[-1] * 65, u=np.zeros((1, 66)))
refuse(INVALID, t, par=None)
refuse(INVALID, t, par=[-1, 1, 0, 0, 0])
refuse(INVALID, d, p=z(17 * (rows + 1) * V), q=z(17 * rows * V), tok=np.zeros((17, rows), int), u=np.zeros((17, rows + 1)))
""",
    "null": """
L = load()
o = (C.c_void_p * 3)()
r = C.byref
def st(name, *a):
    launches()
    rc = getattr(L, "scry_hip_" + name)(*a)
    assert rc == INVALID, (name, rc)
    assert L.scry_hip_last_error()
    assert not launches()
one = (C.c_int32 * 1)(0)
h1 = (C.c_void_p * 1)(c.h)
n1 = (C.c_void_p * 1)(None)
st("buf_dlpack", q.h, None, 0, None)
st("buf_dlpack", None, None, 0, r(C.c_void_p()))
st("buf_dlpack", half.h, None, 0, r(C.c_void_p()))
st("qk_norm_rope", None, 1, rows, one, None, nq, nkv, hd, fr.h, None, None, 1e-5, 1.0, r(C.c_void_p()), r(C.c_void_p()), r(C.c_void_p()))
st("qk_norm_rope", qkv.h, 1, rows, None, None, nq, nkv, hd, fr.h, None, None, 1e-5, 1.0, r(C.c_void_p()), r(C.c_void_p()), r(C.c_void_p()))
st("qk_norm_rope", qkv.h, 1, rows, one, None, nq, nkv, hd, fr.h, None, None, 1e-5, 1.0, r(C.c_void_p()), None, r(C.c_void_p()))
st("kv8_new", ms, nkv, hd, None)
st("kv8_write", None, 1, one, rows, k.h, k.h)
st("kv8_write", n1, 1, one, rows, k.h, k.h)
st("kv8_write", h1, 1, None, rows, k.h, k.h)
st("kv8_write", h1, 1, one, rows, k.h, None)
st("kv8_read", h1, 1, one, rows, r(C.c_void_p()), None)
st("kv8_read", None, 1, one, rows, r(C.c_void_p()), r(C.c_void_p()))
st("kv8_keep", h1, 1, one, None, 1)
long = (C.c_int64 * 1)(1)
st("kv8_keep", None, 1, one, long, 1)
st("kv8_keep", n1, 1, one, long, 1)
st("tree_attention", q.h, None, n1, 1, one, rows, None, nq, nkv, hd, 0.1, r(C.c_void_p()))
st("tree_attention", q.h, n1, n1, 1, one, rows, None, nq, nkv, hd, 0.1, r(C.c_void_p()))
st("tree_attention", q.h, (C.c_void_p * 1)(kc.h), (C.c_void_p * 1)(vc.h), 1, one, rows, None, nq, nkv, hd, 0.1, None)
st("kv8_tree_attention", q.h, n1, 1, one, rows, None, nq, 0.1, r(C.c_void_p()))
st("kv8_tree_attention", q.h, h1, 1, one, rows, None, nq, 0.1, None)
assert L.scry_hip_kv8_free(None) == 0
t1, u1, o1 = (C.c_int64 * 1)(0), (C.c_double * 2)(0, 0), (C.c_int64 * 1)()
p2, p1 = z(2), z(1)
st("verify_draft", p2.h, p1.h, None, None, u1, 1, 1, 1, o1, o1)
st("verify_draft", p2.h, p1.h, t1, None, None, 1, 1, 1, o1, o1)
st("verify_draft", p2.h, None, t1, None, u1, 1, 1, 1, o1, o1)
st("verify_draft", p2.h, p1.h, t1, None, u1, 1, 1, 1, None, o1)
st("verify_tree", p2.h, t1, None, u1, 1, 1, 1, o1, o1, o1)
st("verify_tree", p2.h, t1, (C.c_int64 * 1)(-1), u1, 1, 1, 1, None, o1, o1)
""",
}


@pytest.mark.parametrize("op", list(CALLS))
def test_refusals(fake_hip, op):
    fake_hip(PRE + CALLS[op])


@pytest.mark.parametrize("call", ["B.qk_norm_rope(qkv, [0], rows, nq, nkv, hd, fr)", "B.kv8_read([c], [0], rows)",
                                  "B.tree_attention(q, [kc], [vc], [50], rows, nq, nkv, hd, 0.1)",
                                  "B.kv8_tree_attention(q, [c], [50], rows, nq, 0.1)", "B.kv8_write([c], k, k, [0], rows)",
                                  "B.kv8_keep([c], [0], [[1]])"])
def test_refused_launches_are_errors(fake_hip, call):
    fake_hip(PRE + f"""
{call}
F.fake_refuse(1)
try:
    {call}
except E.ScryHipError as e:
    assert e.code == 2, str(e)
else:
    raise AssertionError("not refused")
F.fake_refuse(0)
{call}
""")


def test_views_hold_their_storage(fake_hip):
    fake_hip(PRE + """
import gc
a = z(1 << 20)
used = F.fake_used()
caps = [a.__dlpack__(stream=-1) for _ in range(3)]
a.free()
b = z(1 << 20)  # another block: the views hold the first
assert F.fake_used() > used
del caps
gc.collect()
used = F.fake_used()
again = z(1 << 20)  # the first
assert F.fake_used() == used
""")


def test_no_memory(fake_hip):
    fake_hip(PRE + """
F.fake_limit(F.fake_used() + (1 << 20))
refuse(OOM, B.kv8_new, 1 << 20, nkv, hd)
F.fake_limit(1 << 40)
B.kv8_new(1 << 20, nkv, hd)
""")


def test_calls_before_init_fail_cleanly():
    import ctypes

    import esolearn_amd as E
    from esolearn_amd import _lib

    n = ctypes.c_int()
    _lib.call("scry_hip_device_count", ctypes.byref(n))
    if n.value > 0:
        pytest.skip("a GPU is present; the no-device path is not reachable")
    with pytest.raises(E.ScryHipError) as ei:
        E.HipBackend.kv8_new(8, 1, 4)
    assert ei.value.code == 4  # SCRY_ERR_NOT_INIT

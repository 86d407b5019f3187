"""What cross_attend, rope_table, rope_rows and groupnorm refuse, checked
without a GPU: every refusal comes before anything is queued."""
import ctypes
import math

import numpy as np
import pytest


@pytest.fixture(scope="module")
def hip():
    import sam3_hip
    sam3_hip.lib()
    return sam3_hip


class Model:
    """A model on a backend that was never opened: the checks need no more."""

    def __init__(self, hip):
        self._b = hip.HipbBackend()
        self.m = hip.SamModel()
        self.m.hip = ctypes.pointer(self._b)

    @property
    def ptr(self):
        return ctypes.byref(self.m)


BASE = 1 << 40     # addresses that are only compared


def mem(hip, n, dt=0, at=0):
    return hip.borrow(BASE + at, n * (4 if dt == 0 else 2), dt)


def cross(hip, **kw):
    d = dict(nb=2, heads=4, kv_heads=2, hd=32, Nq=5, Nk=7)
    t = kw.pop("dt", 0)
    ops = {n: hip.bmat(mem(hip, 100000, t, at), 0, 128, 128 * 8, 32)
           for n, at in (("Q", 0), ("K", 1 << 20), ("V", 2 << 20), ("O", 3 << 20))}
    rest = {}
    for n, v in kw.items():
        (ops if n in ops else d if n in d else rest)[n] = v
    hip.cross_attend(Model(hip), d["nb"], d["heads"], d["kv_heads"], d["hd"], d["Nq"], d["Nk"],
                     ops["Q"], ops["K"], ops["V"], ops["O"], **rest)


@pytest.mark.parametrize("kw,msg", [
    (dict(heads=3), "invalid shape"), (dict(hd=0), "invalid shape"),
    (dict(hd=257), "invalid shape"), (dict(nb=-1), "invalid shape"),
    (dict(Nq=-1), "invalid shape"), (dict(Nk=-1), "invalid shape"),
    (dict(kv_heads=0), "invalid shape"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=math.inf), "scale"),
    (dict(scale=math.nan), "scale"),
])
def test_cross_shapes(hip, kw, msg):
    with pytest.raises(hip.Sam3HipError, match="cross_attend: .*" + msg):
        cross(hip, **kw)


def test_cross_operands(hip):
    def bad(msg, **kw):
        with pytest.raises(hip.Sam3HipError, match="cross_attend: .*" + msg):
            cross(hip, **kw)

    b = hip.bmat
    bad("element type", K=b(mem(hip, 100000, 1, 1 << 20), 0, 128, 1024, 32))
    bad("operand Q reaches", Q=b(mem(hip, 1500), 0, 128, 1024, 32))
    bad("operand K reaches", K=b(mem(hip, 100, 0, 1 << 20), 0, 128, 1024, 32))
    bad("negative offset", V=b(mem(hip, 100000, 0, 2 << 20), -1, 128, 1024, 32))
    bad("ld 16 < 32", Q=b(mem(hip, 100000), 0, 16, 1024, 32))
    bad("without a buffer", O=b(None, 0, 128, 1024, 32))
    bad("writes elements twice", O=b(mem(hip, 100000, 0, 3 << 20), 0, 128, 0, 32))
    bad("writes elements twice", O=b(mem(hip, 100000, 0, 3 << 20), 0, 128, 1024, 16))
    bad("writes elements twice", O=b(mem(hip, 100000, 0, 3 << 20), 0, 64, 1024, 32))
    bad("O overlaps Q", O=b(mem(hip, 100000, 0, 64), 0, 128, 1024, 32))
    bad("O overlaps V", O=b(mem(hip, 100000, 0, 2 << 20), 0, 128, 1024, 32))
    bad("klen", klen=mem(hip, 1, 0, 5 << 20))
    bad("qlen", qlen=mem(hip, 1, 0, 5 << 20))
    bad("kmask", kmask=mem(hip, 3, 0, 5 << 20))
    bad("16 MiB apart", Nk=2, nb=1, kv_heads=1,
        K=b(mem(hip, 1 << 24, 0, 1 << 30), 0, (4 << 20) + 4, 0, 0))


def test_cross_workspace(hip):
    m = Model(hip)
    # Without a device the library counts 256 compute units.
    n = hip.cross_attend_ws(m, 1, 8, 8, 64, 1, 4096, 1)
    assert n > 0 and hip.cross_attend_ws(m, 0, 8, 8, 64, 1, 4096, 1) == 0
    assert hip.cross_attend_ws(m, 64, 32, 32, 64, 4096, 4096, 1) == 0
    with pytest.raises(hip.Sam3HipError, match="cross_attend_ws: unknown element type"):
        hip.cross_attend_ws(m, 1, 8, 8, 64, 1, 4096, 3)
    with pytest.raises(hip.Sam3HipError, match="workspace"):
        cross(hip, nb=1, heads=1, kv_heads=1, Nq=1, Nk=4000,
              K=hip.bmat(mem(hip, 4000 * 128, 0, 1 << 24), 0, 128, 0, 0),
              V=hip.bmat(mem(hip, 4000 * 128, 0, 1 << 26), 0, 128, 0, 0),
              ws=mem(hip, 4, 0, 1 << 30))


def test_cross_too_many_rows(hip):
    with pytest.raises(hip.Sam3HipError, match="too many rows"):
        cross(hip, nb=1 << 20, heads=8, kv_heads=8)
    with pytest.raises(hip.Sam3HipError, match="too many rows"):
        cross(hip, nb=64, heads=64, kv_heads=64, Nq=1 << 20)
    with pytest.raises(hip.Sam3HipError, match="too many rows or keys"):
        cross(hip, Nk=(1 << 30) + 1)


def test_cross_overlaps(hip):
    """Whatever the call writes lies apart from whatever it reads."""
    o = hip.bmat(mem(hip, 100000, 0, 3 << 20), 0, 128, 1024, 32)
    for n, k in (("qlen", 8), ("klen", 8), ("kmask", 14)):
        with pytest.raises(hip.Sam3HipError, match="cross_attend: O overlaps " + n):
            cross(hip, O=o, **{n: mem(hip, k, 0, (3 << 20) + 4096)})
    # Few rows over many keys: split, with sums in ws.
    q = hip.bmat(mem(hip, 100000), 0, 128, 0, 0)
    k = hip.bmat(mem(hip, 4000 * 128, 0, 1 << 24), 0, 128, 0, 0)
    v = hip.bmat(mem(hip, 4000 * 128, 0, 1 << 26), 0, 128, 0, 0)
    o = hip.bmat(mem(hip, 100000, 0, 1 << 28), 0, 128, 0, 0)
    for n, at in (("Q", 0), ("K", 1 << 24), ("V", 1 << 26), ("O", 1 << 28)):
        with pytest.raises(hip.Sam3HipError, match=f"cross_attend: {n} overlaps ws"):
            cross(hip, nb=1, heads=1, kv_heads=1, Nq=1, Nk=4000, Q=q, K=k, V=v, O=o,
                  ws=mem(hip, 1 << 20, 0, at))
    # Columns of one matrix that meet (8 of them), on either side and around its end.
    for at, other in ((0, 24), (24, 0), (104, 0)):
        buf = mem(hip, 100000, 0, 8 << 20)
        with pytest.raises(hip.Sam3HipError, match="O overlaps Q"):
            cross(hip, heads=1, kv_heads=1, Q=hip.bmat(buf, at, 128, 1024, 0),
                  O=hip.bmat(buf, other if at != 104 else 128 * 8, 128, 1024, 0))


def test_other_overlaps(hip):
    x = hip.bmat(mem(hip, 10000), 0, 64, 640, 0)
    y = hip.bmat(mem(hip, 10000, 0, 1 << 20), 0, 64, 640, 0)
    far = mem(hip, 10000, 0, 1 << 24)
    inside = mem(hip, 10000, 0, (1 << 20) + 1024)

    def bad(msg, f, *a, **kw):
        with pytest.raises(hip.Sam3HipError, match=msg):
            f(Model(hip), *a, **kw)

    bad("rope_rows: Y overlaps table", hip.rope_rows, 2, 1, 9, 64, 64, 0, x, y, inside, 9)
    bad("rope_rows: Y overlaps pos", hip.rope_rows, 2, 1, 9, 64, 64, 0, x, y, far, 9, pos=inside)
    bad("rope_rows: too many heads", hip.rope_rows, 2, 1 << 30, 9, 64, 64, 0, x, y, far, 9)
    bad("rope_table: table overlaps pos", hip.rope_table, far, 9,
        mem(hip, 100, 0, (1 << 24) + 64), 64)
    bad("groupnorm: Y overlaps g", hip.groupnorm, 2, 9, 64, 8, x, y, g=inside, b=far)
    bad("groupnorm: Y overlaps b", hip.groupnorm, 2, 9, 64, 8, x, y, g=far, b=inside)
    big = hip.bmat(mem(hip, 1 << 20), 0, 64, 0, 0)
    out = hip.bmat(mem(hip, 1 << 20, 0, 1 << 26), 0, 64, 0, 0)
    for n, at in (("X", 0), ("Y", 1 << 26)):
        bad(f"groupnorm: {n} overlaps ws", hip.groupnorm, 1, 1 << 14, 64, 8, big, out,
            ws=mem(hip, 1 << 20, 0, at))
    bad("rope_rows: Y overlaps X", hip.rope_rows, 2, 1, 9, 64, 32, 0, hip.bmat(far, 0, 128, 1280, 0),
        hip.bmat(far, 32, 128, 1280, 0), mem(hip, 1000), 9)


def test_empty_calls_queue_nothing(hip):
    cross(hip, nb=0)
    cross(hip, Nq=0)
    m = Model(hip)
    t = mem(hip, 1000)
    hip.rope_table(m, t, 0)
    x = hip.bmat(mem(hip, 1000), 0, 8, 0, 0)
    hip.rope_rows(m, 0, 1, 4, 8, 8, hip.ROPE_PAIRS, x, x, t, 4)
    hip.rope_rows(m, 1, 1, 0, 8, 8, hip.ROPE_PAIRS, x, x, t, 4)
    hip.groupnorm(m, 0, 4, 8, 2, x, x)
    hip.groupnorm(m, 1, 0, 8, 2, x, x)


@pytest.mark.parametrize("kw", [
    dict(rot=0), dict(rot=7), dict(rot=514), dict(npos=-1), dict(theta=0.0),
    dict(theta=math.inf), dict(theta=math.nan), dict(W=-1), dict(W=8, rot=6),
])
def test_table_shapes(hip, kw):
    d = dict(npos=4, rot=8, W=0, theta=100.0)
    d.update(kw)
    with pytest.raises(hip.Sam3HipError, match="rope_table: invalid npos"):
        hip.rope_table(Model(hip), mem(hip, 10000), d["npos"], None, d["rot"], d["W"], d["theta"])


@pytest.mark.parametrize("kw", [
    dict(kind=4), dict(kind=-1), dict(kind=1, factor=0.5), dict(kind=1, factor=math.nan),
    dict(kind=2, factor=math.inf), dict(kind=3, factor=2.0, orig=0, beta_fast=32.0, beta_slow=1.0),
    dict(kind=3, factor=2.0, orig=64, beta_fast=1.0, beta_slow=1.0),
    dict(kind=3, factor=2.0, orig=64, beta_fast=math.inf, beta_slow=1.0),
])
def test_table_scaling(hip, kw):
    with pytest.raises(hip.Sam3HipError, match="rope_table: invalid scaling"):
        hip.rope_table(Model(hip), mem(hip, 10000), 4, None, 8, scale=hip.RopeScale(**kw))


def test_table_buffers(hip):
    m = Model(hip)
    with pytest.raises(hip.Sam3HipError, match="rope_table: invalid scaling"):
        hip.rope_table(m, mem(hip, 10000), 4, None, 8, W=2,
                       scale=hip.RopeScale(kind=1, factor=2.0))
    with pytest.raises(hip.Sam3HipError, match="rope_table: table .* holds 31 elements, 32"):
        hip.rope_table(m, mem(hip, 31), 4, None, 8)
    with pytest.raises(hip.Sam3HipError, match="rope_table: table .* element type"):
        hip.rope_table(m, mem(hip, 100, 1), 4, None, 8)
    with pytest.raises(hip.Sam3HipError, match="rope_table: pos"):
        hip.rope_table(m, mem(hip, 100), 4, mem(hip, 3, 0, 1 << 20), 8)
    with pytest.raises(hip.Sam3HipError, match="8-byte aligned"):
        hip.rope_table(m, mem(hip, 100, 0, 4), 4, None, 8)


def test_rope_rows_refusals(hip):
    m = Model(hip)
    b = hip.bmat
    t = mem(hip, 64 * 16, 0, 1 << 30)
    x, y = b(mem(hip, 10000), 0, 64, 320, 16), b(mem(hip, 10000, 0, 1 << 20), 0, 64, 320, 16)

    def bad(msg, nb=2, heads=4, rows=5, hd=16, rot=16, layout=0, X=x, Y=y, T=t, npos=64, pos=None,
            pos0=0):
        with pytest.raises(hip.Sam3HipError, match="rope_rows: .*" + msg):
            hip.rope_rows(m, nb, heads, rows, hd, rot, layout, X, Y, T, npos, pos, pos0)

    bad("invalid shape", rot=18)
    bad("invalid shape", rot=3)
    bad("invalid shape", rot=0)
    bad("invalid shape", layout=2)
    bad("invalid shape", npos=0)
    bad("invalid shape", pos0=-1)
    bad("invalid shape", heads=0)
    bad("operand X reaches", X=b(mem(hip, 600), 0, 64, 320, 16))
    bad("operand Y reaches", Y=b(mem(hip, 600, 0, 1 << 20), 0, 64, 320, 16))
    bad("one element type", Y=b(mem(hip, 10000, 1, 1 << 20), 0, 64, 320, 16))
    bad("writes elements twice", Y=b(mem(hip, 10000, 0, 1 << 20), 0, 64, 320, 8))
    bad("writes elements twice", Y=b(mem(hip, 10000, 0, 1 << 20), 0, 64, 100, 16))
    bad("overlaps X", Y=b(mem(hip, 10000), 16, 64, 320, 16))
    bad("table", T=mem(hip, 1023, 0, 1 << 30))
    bad("pos", pos=mem(hip, 9, 0, 1 << 31))
    bad("8-byte aligned", T=mem(hip, 1024, 0, (1 << 30) + 4))


def test_groupnorm_refusals(hip):
    m = Model(hip)
    b = hip.bmat
    x, y = b(mem(hip, 10000), 0, 32, 320, 0), b(mem(hip, 10000, 0, 1 << 20), 0, 32, 320, 0)

    def bad(msg, nb=2, rows=10, C=32, groups=4, X=x, Y=y, g=None, be=None, eps=1e-5, act=0,
            ws=None):
        with pytest.raises(hip.Sam3HipError, match="groupnorm: .*" + msg):
            hip.groupnorm(m, nb, rows, C, groups, X, Y, g, be, eps, act, ws)

    bad("invalid shape", groups=5)
    bad("invalid shape", groups=0)
    bad("invalid shape", C=0)
    bad("invalid shape", nb=70000)
    bad("invalid shape", rows=-1)
    bad("invalid shape", C=8192, groups=8192)
    bad("invalid act", act=4)
    bad("invalid act", act=-1)
    bad("invalid act", eps=-1.0)
    bad("invalid act", eps=math.nan)
    bad("operand X reaches", X=b(mem(hip, 600), 0, 32, 320, 0))
    bad("operand Y reaches", Y=b(mem(hip, 600, 0, 1 << 20), 0, 32, 320, 0))
    bad("one element type", Y=b(mem(hip, 10000, 2, 1 << 20), 0, 32, 320, 0))
    bad("writes elements twice", Y=b(mem(hip, 10000, 0, 1 << 20), 0, 32, 300, 0))
    bad("overlaps X", Y=b(mem(hip, 10000), 8, 32, 320, 0))
    bad("overlaps X", Y=b(mem(hip, 10000), 0, 64, 640, 0))
    bad("g <", g=mem(hip, 31, 0, 1 << 30))
    bad("b <", be=mem(hip, 31, 0, 1 << 30))
    big = 1 << 20
    bad("workspace", nb=1, rows=big // 32, X=b(mem(hip, big), 0, 32, 0, 0),
        Y=b(mem(hip, big, 0, 1 << 24), 0, 32, 0, 0), ws=mem(hip, 4, 0, 1 << 30))
    assert hip.groupnorm_ws(m, 1, big // 32, 32, 4, 0) > 0
    assert hip.groupnorm_ws(m, 1, 4, 32, 4, 0) == 0


def test_silu_is_groupnorms_alone(hip):
    m = Model(hip)
    t = mem(hip, 1024)
    with pytest.raises(hip.Sam3HipError, match="layernorm"):
        hip.layernorm(m, 4, 32, t, t, t, t, 1e-5, hip.ACT_SILU)


def test_borrowed_handle(hip):
    b = hip.borrow(0x1000, 64, hip.BF16, "states").contents
    assert (b.ptr, b.bytes, b.dtype, b.what) == (0x1000, 64, hip.BF16, b"states")


def test_structs_match_header(hip):
    import os
    import re
    src = open(os.path.join(os.path.dirname(hip.HERE), "include", "sam3_hip.h")).read()
    body = re.search(r"struct rope_scale \{(.*?)\};", src, re.S).group(1)
    names = re.findall(r"([A-Za-z_]+)\s*[,;]", body)
    assert [f[0] for f in hip.RopeScale._fields_] == names
    for n in ("ROPE_PAIRS", "ROPE_HALVES", "ROPE_PLAIN", "ROPE_LINEAR", "ROPE_NTK", "ROPE_YARN",
              "ACT_SILU"):
        assert int(re.search(r"#define %s (\d+)" % n, src).group(1)) == getattr(hip, n)


def test_bounds_count_roundings():
    """The bound of the attention's tests on values worked by hand: float
    products of one key leave only the roundings named in it."""
    import seq_common as sc
    q = np.ones((1, 1, 1, 2))
    o, av, top, prod = sc.cross(q, q, 3 * q, np.ones((1, 1), bool), 1.0)
    assert (o == 3).all() and (av == 3).all() and (top == 2).all() and (prod == 2).all()
    lim = sc.cross_bound(o, av, top, prod, 2, 1, sc.F32, 3 * q)
    assert (lim < 3 * 1e-5).all() and (lim > 3 * 2.0 ** -24).all()
